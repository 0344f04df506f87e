"""Operators of the decoder training step as HIP kernels for MI355X.

    attention(q, k, v)            self-attention over grouped heads
    token_logprobs(logits, ids)   log p(token), entropy, alternatives
    residual_norm(x, branch, w)   residual sum and the RMS norm of it

All three are differentiable (first derivatives, backward mode), run on the current stream of
their tensors' device, allocate what they return and nothing that outlives the
call, give the same bits for the same inputs, and can be captured into a graph
(a backward pass, as always with torch, while no eager graph of its leaves lives).
They are operators of torch's dispatcher (torch.ops.sofa_model), which its tracers
record.  They need tensors on a GPU: there is no other path, and a missing library is an
error.  Wrong arguments raise TypeError (types) or ValueError (shapes, values).

`Llama(kernels="hip")` and `python -m sofa_amd.workloads.llama --kernels hip`
run the decoder on them, under bfloat16 autocast or with bfloat16 weights.  The
kernels are in native/hip/model.
"""

from __future__ import annotations

import importlib.util
import math
import os
from typing import NamedTuple, Optional, Tuple

import torch

_TYPES = (torch.float32, torch.bfloat16, torch.float16)

MAX_HEAD_DIM = 128
MAX_TOKENS = 1 << 24
_MAX_BLOCKS = (1 << 24) - 1  # 128 tokens of one head each
MAX_TOP = 32
MAX_NORM_DIM = 16384
_MAX_GATES = 1 << 21
MAX_VOCAB = 1 << 30

_module = None


def _ops():
    """The binding of the kernels to torch."""
    global _module
    if _module is None:
        path = os.path.join(
            os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
            "native", "lib", "sofa_model.so",
        )
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is not built: run python -m sofa_amd.native.build")
        spec = importlib.util.spec_from_file_location("sofa_model", path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        _module = module
    return _module


def _on_gpu(what: str, first: torch.Tensor, **others: Optional[torch.Tensor]) -> None:
    if first.device.type != "cuda":
        raise ValueError(f"{what}: tensors on a GPU are needed, got one on {first.device}")
    for name, t in others.items():
        if t is not None and t.device != first.device:
            raise ValueError(f"{what}: {name} is on {t.device}, not on {first.device}")


# ------------------------------------------------------------------ attention
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
    128, and computed as if it were 64 or 128; any strides (rows that are not dense
    or not at multiples of 16 bytes are copied first).  scale is above 0 (1e-18 to 1e18), 1 / sqrt(dim) if not given.

    causal: token i sees tokens 0..i, otherwise all.  lengths: int32 (batch,),
    the valid tokens at the front of each sequence, taken as within 0..tokens;
    what stands behind them is never used, whatever it is, and its results and
    gradients are zeros.  Valid tokens have to be finite, the later ones that a
    causal mask hides included.

    float16 is refused: the gradient of a score, which the products of the
    backward pass take in the inputs' type, is below float16's smallest normal
    value in long sequences.

    Scores are sums of 32 bits: one of size s is off by some 2^-24 s, and its
    probability by that share.  The products of probabilities, and in rows that see
    more than 256 keys those of the scores' gradients, take them rounded to bfloat16;
    a score's gradient is good to 2^-17 of the gradient of its probability.

    Returns (batch, heads, tokens, dim), laid out as (batch, tokens, heads, dim).
    For a backward pass q, k, v and twice the size of the result are kept.
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
    if tokens > MAX_TOKENS or batch * heads * -(-tokens // 128) > _MAX_BLOCKS:
        raise ValueError(f"attention: {tuple(q.shape)} is too large")
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    elif not 1e-18 <= scale <= 1e18:
        raise ValueError(f"attention: scale has to be within 1e-18..1e18, got {scale}")
    if lengths is not None:
        if lengths.dtype != torch.int32:
            raise TypeError(f"attention: lengths has to be int32, got {lengths.dtype}")
        if lengths.shape != (batch,):
            raise ValueError(f"attention: lengths has to be ({batch},), got {tuple(lengths.shape)}")
    _on_gpu("attention", q, k=k, v=v, lengths=lengths)
    if q.numel() == 0:
        return q + 0 * (k.sum() + v.sum())  # no tokens: empty, and still part of the graph
    return _ops().attention(q, k, v, lengths, scale, causal)


# ------------------------------------------------------------------ token log probabilities
class TokenLogprobs(NamedTuple):
    """logprob and entropy (differentiable) have the tokens' shape; top_ids and
    top_logprobs have one more axis of `top`, most likely first, or are None."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    top_ids: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]


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
    outside 0..vocab-1 has log probability NaN, and NaN for a gradient that passes
    through it.  Logits of -inf are tokens that are not allowed.  A row without an
    allowed token has log probability -inf, entropy 0 and gradient 0; one with a
    NaN or +inf has NaN throughout, in its gradient too where one comes in.
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
    if top:
        return TokenLogprobs(*_ops().token_logprobs_top(logits, tokens, top, ignore_index))
    return TokenLogprobs(*_ops().token_logprobs(logits, tokens, ignore_index), None, None)


# ------------------------------------------------------------------ residual norm
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
    if not 0 <= eps <= 1e30:
        raise ValueError(f"residual_norm: eps has to be within 0..1e30, got {eps}")
    if not abs(scale) <= 1e30:
        raise ValueError(f"residual_norm: scale has to be within -1e30..1e30, got {scale}")
    if gate is not None and gate.numel() // dim > _MAX_GATES:
        raise ValueError(f"residual_norm: {gate.numel() // dim} gates are too many")
    if x.numel() // dim > 2**31 - 1:
        raise ValueError(f"residual_norm: {x.numel() // dim} rows are too many")
    _on_gpu("residual_norm", x, branch=branch, weight=weight, post_weight=post_weight, gate=gate)
    if x.numel() == 0:  # empty, and still part of the graph
        r = x
        for t in (branch, post_weight, gate):
            r = r if t is None else r * t.to(x.dtype)
        return (x if branch is None else r), (r * weight.to(x.dtype)).to(out_dtype)
    if branch is None:
        return x, _ops().rms_norm(x, weight, eps, out_dtype)
    return _ops().residual_norm(x, branch, weight, post_weight, gate, scale, eps, out_dtype)
