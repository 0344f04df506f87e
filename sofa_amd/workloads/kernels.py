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
import struct
from typing import NamedTuple, Optional, Tuple

import torch

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

MAX_HEAD_DIM = 128
MAX_TOKENS = 1 << 24
MAX_TOP = 32
_MAX_TOKEN_STRIDE = 1 << 24  # elements
MAX_NORM_DIM = 16384
MAX_VOCAB = 1 << 30

# The argument structures of the C entries, packed in one call each: pointers,
# then 64-bit, 32-bit floating and 32-bit whole numbers, in the order of their
# declarations in native/hip/model.  "0q" pads the end as C does.
_ATTENTION = struct.Struct("14P24qf8i0q")
_LOGPROBS = struct.Struct("13P11q6i0q")
_NORM = struct.Struct("16P2q2f9i0q")

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
            entry.argtypes, entry.restype = [ctypes.c_char_p], ctypes.c_int
        _lib_handle = lib
    return _lib_handle


def _call(name: str, args: bytes) -> None:
    status = getattr(_lib_handle or _lib(), name)(args)
    if status:
        what = "bad argument" if status < 0 else f"HIP error {status}"
        raise RuntimeError(f"{name} failed: {what}")


# a torch.cuda.Stream object for each call would cost as much as the launch
_stream = torch._C._cuda_getCurrentRawStream


def _once(backward):
    """A backward pass that is itself recorded only to refuse a second one."""
    recorded = torch.autograd.function.once_differentiable(backward)

    def either(ctx, *grads):
        return (recorded if torch.is_grad_enabled() else backward)(ctx, *grads)

    return either


def _on_gpu(what: str, first: torch.Tensor, **others: Optional[torch.Tensor]) -> None:
    if first.device.type != "cuda":
        raise ValueError(f"{what}: tensors on a GPU are needed, got one on {first.device}")
    for name, t in others.items():
        if t is not None and t.device != first.device:
            raise ValueError(f"{what}: {name} is on {t.device}, not on {first.device}")


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _recorded(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether autograd will ask for a backward pass."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ------------------------------------------------------------------ attention
def _rows16(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy, with dense rows that start at multiples of 16 bytes and are
    not further apart than the kernels' offsets within a tile reach."""
    a, b, c, dense = t.stride()
    if dense == 1 and c <= _MAX_TOKEN_STRIDE and t.data_ptr() % 16 == 0 and (a | b | c) % 8 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _token_major(like: torch.Tensor) -> torch.Tensor:
    """(batch, heads, tokens, dim) laid out as (batch, tokens, heads, dim): what
    the projection behind it reads as one matrix without a copy."""
    batch, heads, tokens, dim = like.shape
    return like.new_empty_strided(like.shape, (tokens * heads * dim, dim, heads * dim, 1))


_NO_STRIDES = (0,) * 12


def _attention_forward(q, k, v, lengths, scale, causal, recorded):
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    batch, heads, tokens, dim = q.shape
    o, o_low, lse = _token_major(q), None, None
    if recorded:
        o_low, lse = _token_major(q), q.new_empty((batch, heads, tokens), dtype=torch.float32)
    strides = (*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *o.stride()[:3])
    device = q.device.index
    _call("sofa_attention_forward", _ATTENTION.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _ptr(o_low), _ptr(lse), _ptr(lengths),
        0, 0, 0, 0, 0, 0, _stream(device), *strides, *_NO_STRIDES, scale,
        batch, heads, k.shape[1], tokens, dim, causal, 1, device))
    return q, k, v, o, o_low, lse


def _key_parts(batch: int, heads: int, kv_heads: int, tokens: int, dim: int, causal: bool) -> int:
    """Workgroups that share the rows behind one block of 128 keys. Two fit a
    compute unit, so 512 fill the card; under a causal mask the blocks differ in
    work and twice as many even it out (8192 tokens, 8 key heads of 128: 1.15 ms
    with two parts, 1.71 with one). Parts cost a pass over their sums, and one
    of less than four steps gains nothing."""
    groups = batch * kv_heads * -(-tokens // 128)
    steps = -(-tokens // (64 if dim <= 64 else 32)) * (heads // kv_heads) // (2 if causal else 1)
    return max(1, min(8, -(-(1024 if causal else 512) // groups), steps // 4))


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, scale, causal):
        q, k, v, o, o_low, lse = _attention_forward(q, k, v, lengths, scale, causal, True)
        ctx.save_for_backward(q, k, v, o, o_low, lse, lengths)
        ctx.scale, ctx.causal = scale, causal
        return o

    @staticmethod
    @_once
    def backward(ctx, dout):
        q, k, v, o, o_low, lse, lengths = ctx.saved_tensors
        dout = _rows16(dout)
        delta = torch.empty_like(lse)
        dq, dk, dv = _token_major(q), _token_major(k), _token_major(v)
        batch, heads, tokens, dim = q.shape
        kv_heads, device = k.shape[1], q.device.index
        parts = _key_parts(batch, heads, kv_heads, tokens, dim, ctx.causal)
        partial = q.new_empty((parts, 2, *k.shape), dtype=torch.float32) if parts > 1 else None
        _call("sofa_attention_backward", _ATTENTION.pack(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), o_low.data_ptr(), lse.data_ptr(), _ptr(lengths),
            dout.data_ptr(), delta.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
            _ptr(partial), _stream(device),
            *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *o.stride()[:3],
            *dout.stride()[:3], *dq.stride()[:3], *dk.stride()[:3], *dv.stride()[:3], ctx.scale,
            batch, heads, kv_heads, tokens, dim, ctx.causal, parts, device))
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
    if t.is_contiguous():
        width = t.shape[-1] if axes < t.dim() else 1
        return t.numel() // width, 0, width
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
    """(parts, part_size): a row goes to one workgroup where there are rows for
    every compute unit, which then read all that memory gives; below that it is
    cut into parts."""
    step = 2048  # what a workgroup of 256 threads reads at a time
    parts = max(1, min(64, -(-256 // rows), -(-vocab // step)))
    size = -(-vocab // (parts * step)) * step
    return -(-vocab // size), size


def _logprob_forward(logits, tokens, top, ignore_index):
    axes, rows, vocab = tokens.dim(), tokens.numel(), logits.shape[-1]
    split = _two_level(logits, axes) if logits.stride(-1) == 1 else None
    if split is None:
        logits = logits.contiguous()
        split = rows, 0, vocab
    tokens, *token_strides = _same_split(split[0], rows, tokens, axes)
    shape = tokens.shape
    logprob, entropy, lse = (logits.new_empty(shape, dtype=torch.float32) for _ in range(3))
    parts, part_size = _logprob_split(rows, vocab)
    ids = values = part_sums = part_top = None
    if top:
        ids = tokens.new_empty((*shape, top))
        values = logits.new_empty((*shape, top), dtype=torch.float32)
    if parts > 1:
        part_sums = logits.new_empty((rows, parts, 3), dtype=torch.float32)
        if top:
            part_top = tokens.new_empty((rows, parts, top))
    device = logits.device.index
    _call("sofa_logprob_forward", _LOGPROBS.pack(
        logits.data_ptr(), tokens.data_ptr(), logprob.data_ptr(), entropy.data_ptr(), lse.data_ptr(),
        _ptr(ids), _ptr(values), _ptr(part_sums), _ptr(part_top), 0, 0, 0, _stream(device),
        rows, *split, 0, 0, 0, 0, *token_strides, ignore_index,
        vocab, top, parts, part_size, _TYPES[logits.dtype], device))
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
    @_once
    def backward(ctx, dlogprob, dentropy, _ids, _values):
        if dlogprob is None and dentropy is None:
            return None, None, None, None
        logits, tokens, entropy, lse = ctx.saved_tensors
        axes, rows, vocab = tokens.dim(), tokens.numel(), logits.shape[-1]
        split = _two_level(logits, axes)
        tokens, *token_strides = _same_split(split[0], rows, tokens, axes)
        strides = [0, 0, 0, 0]
        if dlogprob is not None:
            dlogprob, *strides[:2] = _same_split(split[0], rows, dlogprob, axes)
        if dentropy is not None:
            dentropy, *strides[2:] = _same_split(split[0], rows, dentropy, axes)
        dlogits = torch.empty_like(logits, memory_format=torch.contiguous_format)
        parts, part_size = _logprob_split(rows, vocab)
        device = logits.device.index
        _call("sofa_logprob_backward", _LOGPROBS.pack(
            logits.data_ptr(), tokens.data_ptr(), entropy.data_ptr(), entropy.data_ptr(), lse.data_ptr(),
            0, 0, 0, 0, _ptr(dlogprob), _ptr(dentropy), dlogits.data_ptr(), _stream(device),
            rows, *split, *strides, *token_strides, ctx.ignore_index,
            vocab, 0, parts, part_size, _TYPES[logits.dtype], device))
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
def _norm_pack(pointers, x, branch_dtype, y_dtype, weight, post, gate, scale, eps, blocks=0):
    dim = x.shape[-1]
    rows = x.numel() // dim
    group_rows = rows if gate is None else rows * dim // gate.numel()
    device = x.device.index
    return _NORM.pack(
        *pointers, _stream(device), rows, group_rows, eps, scale, dim,
        _TYPES[x.dtype], _TYPES[branch_dtype], _TYPES[y_dtype], _TYPES[weight.dtype],
        0 if post is None else _TYPES[post.dtype], 0 if gate is None else _TYPES[gate.dtype], blocks, device)


def _norm_blocks(rows: int, groups: int, dim: int) -> int:
    """Workgroups of the backward pass that share the rows of one gate. About 512
    fill the card twice; more would only add partial sums."""
    rows //= groups
    return max(1, min(512 // groups, -(-rows // 4) if dim <= 1024 else rows))


def _norm_forward(x, branch, weight, post, gate, scale, eps, out_dtype):
    y = torch.empty_like(x, dtype=out_dtype)
    r = None if branch is None else torch.empty_like(x)
    # without a branch its type only chooses a kernel, and one is built for y's
    _call("sofa_norm_forward", _norm_pack(
        (x.data_ptr(), _ptr(branch), weight.data_ptr(), _ptr(post), _ptr(gate), _ptr(r), y.data_ptr(),
         0, 0, 0, 0, 0, 0, 0, 0),
        x, out_dtype if branch is None else branch.dtype, out_dtype, weight, post, gate, scale, eps))
    return r, y


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, weight, post, gate, scale, eps, out_dtype):
        r, y = _norm_forward(x, branch, weight, post, gate, scale, eps, out_dtype)
        ctx.set_materialize_grads(False)
        ctx.args = scale, eps, out_dtype, None if branch is None else branch.dtype
        # a 32-bit sum is kept, one rounded to 16 bits is computed again
        if branch is not None and x.dtype == torch.float32:
            x = r
            if post is None and gate is None:
                branch = None
        ctx.save_for_backward(x, branch, weight, post, gate)
        return r, y

    @staticmethod
    @_once
    def backward(ctx, dr, dy):
        if dr is None and dy is None:
            return (None,) * 8
        x, branch, weight, post, gate = ctx.saved_tensors
        scale, eps, out_dtype, branch_dtype = ctx.args
        dr, dy = dr if dr is None else dr.contiguous(), dy if dy is None else dy.contiguous()
        _, need_branch, need_weight, need_post, need_gate = ctx.needs_input_grad[:5]
        dx = torch.empty_like(x)
        dbranch = torch.empty_like(x, dtype=branch_dtype) if need_branch else None
        dweight = torch.empty_like(weight) if need_weight else None
        dpost = torch.empty_like(post) if need_post else None
        dgate = torch.empty_like(gate) if need_gate else None
        dim = x.shape[-1]
        groups = 1 if gate is None else gate.numel() // dim
        blocks = _norm_blocks(x.numel() // dim, groups, dim)
        sums = need_weight + need_post + need_gate
        partial = x.new_empty((sums, groups * blocks, dim), dtype=torch.float32) if sums else None
        _call("sofa_norm_backward", _norm_pack(
            (x.data_ptr(), _ptr(branch), weight.data_ptr(), _ptr(post), _ptr(gate), 0, 0,
             _ptr(dr), _ptr(dy), dx.data_ptr(), _ptr(dbranch), _ptr(partial),
             _ptr(dweight), _ptr(dpost), _ptr(dgate)),
            x, branch_dtype or out_dtype, out_dtype, weight, post, gate, scale, eps, blocks))
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
    dense = (t if t is None or t.is_contiguous() else t.contiguous() for t in (x, branch, weight, post_weight, gate))
    args = (*dense, float(scale), float(eps), out_dtype)
    if _recorded(x, branch, weight, post_weight, gate):
        r, y = _ResidualNorm.apply(*args)
    else:
        r, y = _norm_forward(*args)
    return (x if branch is None else r), y
