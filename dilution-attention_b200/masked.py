"""Softmax attention of training steps and prompts whose scores are more than causal.

    softmax_attention(q, k, v, softcap=, slopes=, documents=, prefix=)

    s_ij  = q_i . k_j / sqrt(D)
    c_ij  = softcap * tanh(s_ij / softcap)                  (s_ij without a cap)
    a_ij  = c_ij - slopes_h * |i - j|
    query i sees key j  <=>  (j <= i  or  j < prefix_b)  and  documents_bi = documents_bj >= 0
    out_i = sum_j softmax_j(a_ij over the keys that i sees) v_j

Differentiable in q, k and v.  It stands next to `softmax_attention_forward` (causal, heads of 64, no gradient); a token
or a tree of drafted tokens over a cache has the same scores in `softmax_tree_step`.  Nothing (T x T)-shaped is stored,
tiles of tokens that do not see one another are passed over, and every result repeats bit for bit.
"""

from __future__ import annotations

import contextlib
import math

import torch

from . import _lib
from . import kernels as K

_DIMS = (16, 32, 64, 128)
_INT_MAX = 2 ** 31 - 1
_CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}


def on_device(device):
    """The tensors' device as the current one: launches go to one of its streams."""
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def aligned(x):
    """Contiguous and on a 16-byte boundary."""
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def check_softcap(softcap) -> float:
    """The cap as the kernels take it, 0 for none."""
    if softcap is None:
        return 0.0
    softcap = float(softcap)
    if not 1e-30 <= softcap <= 1e38:
        raise ValueError("softcap must be a number from 1e-30 to 1e38, or None")
    return softcap


def check_slopes(slopes, heads, device):
    """(heads,) fp32 on the device, or None."""
    if slopes is None:
        return None
    if not isinstance(slopes, torch.Tensor):
        slopes = torch.tensor(slopes, dtype=torch.float32, device=device)
    if slopes.shape != (heads,) or not slopes.is_floating_point():
        raise ValueError(f"slopes must be one number for each of the {heads} query heads")
    if slopes.requires_grad:
        raise ValueError("slopes have no gradient here; pass slopes.detach()")
    if slopes.device != device:
        raise ValueError("slopes must be on q's device")
    return slopes.float().contiguous()


def _integers(x, shape, name, device):
    """int32 on the device, in the given shape; anything below 0 is as good as -1 here, and nothing wraps."""
    if not isinstance(x, torch.Tensor) or x.dtype not in (torch.int32, torch.int64) or x.shape != shape:
        raise ValueError(f"{name} must be an int32 or int64 tensor of shape {tuple(shape)}")
    if x.device != device:
        raise ValueError(f"{name} must be on q's device")
    if x.dtype == torch.int64:
        x = x.clamp(-1, _INT_MAX)
    return x.to(torch.int32).contiguous()


def check_heads(q, k, v):
    """(batch, heads, kv_heads, tokens, head size) of q (B, H, T, D) and k, v (B, H_kv, T, D)."""
    if not q.is_cuda:
        raise RuntimeError("softmax attention needs CUDA tensors (no CPU fallback in this backend)")
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError("q, k and v are (batch, heads, tokens, head_dim), k and v of one shape")
    batch, heads, seq, dim = q.shape
    if k.shape[0] != batch or k.shape[2] != seq or k.shape[3] != dim:
        raise ValueError("k and v must have q's batch, tokens and head_dim")
    if k.shape[1] < 1 or heads % k.shape[1]:
        raise ValueError(f"{k.shape[1]} key heads do not divide {heads} query heads")
    if q.dtype not in _CODE or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must be all float32 or all bfloat16")
    if k.device != q.device or v.device != q.device:
        raise ValueError("q, k and v must be on one device")
    if dim not in _DIMS:
        raise ValueError(f"head_dim {dim} not in {_DIMS}")
    return batch, heads, k.shape[1], seq, dim


class _SoftmaxAttention(torch.autograd.Function):
    """Saved for the backward: q, k, v and out as the kernels took them, what out's rounding to bf16 left off, lse, and the
    ranges of the documents' ids."""

    @staticmethod
    def forward(ctx, q, k, v, slopes, documents, prefix, softcap):
        batch, heads, kv_heads, seq, dim = ctx.sizes = (*q.shape[:2], k.shape[1], *q.shape[2:])
        ctx.softcap = softcap
        out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
        if out.numel() == 0:
            return out
        lib = _lib.load()
        train = any(ctx.needs_input_grad[:3])
        q, k, v = (aligned(x) for x in (q, k, v))
        lse = torch.empty(batch, heads, seq, device=q.device, dtype=torch.float32) if train else None
        rest = torch.empty_like(out) if train and q.dtype == torch.bfloat16 else None
        ranges = None
        if documents is not None:
            ranges = torch.empty(lib.dilution_attend_ranges_bytes(batch, seq), device=q.device, dtype=torch.uint8)
        with on_device(q.device):
            _lib.check(lib.dilution_attend_forward(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), _CODE[q.dtype], batch, heads, kv_heads, seq, dim, 1.0 / math.sqrt(dim),
                softcap, K._ptr(slopes), K._ptr(documents), K._ptr(prefix), K._ptr(ranges), out.data_ptr(), K._ptr(rest),
                K._ptr(lse), K._stream(q.device)), "dilution_attend_forward")
        if train:
            ctx.save_for_backward(q, k, v, out, rest, lse, slopes, documents, prefix, ranges)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        batch, heads, kv_heads, seq, dim = ctx.sizes
        if dout.numel() == 0:
            kv = (batch, kv_heads, seq, dim)
            return dout, dout.new_zeros(kv), dout.new_zeros(kv), None, None, None, None
        q, k, v, out, rest, lse, slopes, documents, prefix, ranges = ctx.saved_tensors
        lib = _lib.load()
        dout = aligned(dout)
        dq, dk, dv = (torch.empty(x.shape, device=x.device, dtype=x.dtype) for x in (q, k, v))
        scratch = torch.empty(lib.dilution_attend_scratch_bytes(batch, heads, seq), device=q.device, dtype=torch.uint8)
        with on_device(q.device):
            _lib.check(lib.dilution_attend_backward(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), _CODE[q.dtype], batch, heads, kv_heads, seq, dim, 1.0 / math.sqrt(dim),
                ctx.softcap, K._ptr(slopes), K._ptr(documents), K._ptr(prefix), K._ptr(ranges), out.data_ptr(), K._ptr(rest),
                lse.data_ptr(), dout.data_ptr(), scratch.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), K._stream(q.device)),
                "dilution_attend_backward")
        return dq, dk, dv, None, None, None, None


def softmax_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, softcap: float | None = None,
                      slopes: torch.Tensor | None = None, documents: torch.Tensor | None = None,
                      prefix: torch.Tensor | int | None = None) -> torch.Tensor:
    """Causal softmax attention with capped scores, a distance bias, documents and a prefix (see the module).

    q: (B, H, T, D); k, v: (B, H_kv, T, D) with H_kv dividing H, query head h on key head h // (H / H_kv); all float32
    or all bfloat16, D in {16, 32, 64, 128}, any strides.  Returns (B, H, T, D) in q's dtype.

    softcap: scores go through softcap * tanh(s / softcap), from 1e-30 to 1e38.  slopes: (H,), constants of either sign.  documents: (B, T) int32 or int64
    ids below 2^31; a token sees its own document alone, and one with a negative id (padding) sees and is seen by nothing:
    its output and its gradients are zero, and what its rows hold does not matter.  prefix: (B,) integers or one for all;
    the first `prefix` tokens are seen by every token of their sequence (and document).
    """
    batch, heads, _, seq, _ = check_heads(q, k, v)
    softcap = check_softcap(softcap)
    slopes = check_slopes(slopes, heads, q.device)
    if documents is not None:
        documents = _integers(documents, (batch, seq), "documents", q.device)
    if prefix is not None:
        if isinstance(prefix, int):
            prefix = torch.full((batch,), min(max(prefix, 0), _INT_MAX), device=q.device, dtype=torch.int32)
        prefix = _integers(prefix, (batch,), "prefix", q.device)
    return _SoftmaxAttention.apply(q, k, v, slopes, documents, prefix, softcap)
