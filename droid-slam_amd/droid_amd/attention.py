"""Token operators on keyframe feature maps: position rotation and attention over packed sequences, with their gradients.

A keyframe's feature map ``[h, w]`` is h * w tokens (row by row), a window of keyframes their concatenation, several windows are packed one
behind the other in one tensor ``[rows, heads, head_dim]``.

``qk_norm_rope``      norm of every query and key head and rotation by the token's (keyframe, row, column), one kernel
                      (droid_backends.qk_norm_rope_forward / _backward)
``PackedPlan``        work items of one set of sequence lengths, laid out once on the host
``packed_attention``  softmax attention of the packed queries over the packed keys, grouped heads, all keys / token by token / keyframe by
                      keyframe (droid_backends.attention_forward / attention_backward)

Both are differentiable once.  All work runs on the tensors' device and its current stream; nothing synchronises but the construction of a
PackedPlan (a copy to the device: build it before a graph is captured)."""
import math

import torch

import droid_backends


class PackedPlan:
    """Work items of ``packed_attention`` for sequences of `lengths` query tokens (host integers; 0 is allowed).

    key_lengths    keys of each sequence (default: `lengths`)
    causal_block   0: a token sees every key of its sequence.  1: the keys up to its own, the last token standing at the last key.
                   n: the keys up to the end of its block of n keys (a keyframe of n tokens sees itself and earlier keyframes)
    key_starts     first key row of each sequence (default: packed one behind the other), e.g. the slots of a cache

    Query rows are packed one behind the other from row 0 on.  The plan belongs to its lengths, heads, head_dim and device; it may be used
    by any number of calls, also at once on several streams, and in captured graphs (which it has to outlive)."""

    def __init__(self, lengths, heads, kv_heads, head_dim, key_lengths=None, causal_block=0, key_starts=None, device="cuda"):
        lengths = [int(n) for n in lengths]
        key_lengths = lengths if key_lengths is None else [int(n) for n in key_lengths]
        if key_starts is not None:
            key_starts = [int(n) for n in key_starts]
        items, self.info = droid_backends.attention_plan(lengths, key_lengths, key_starts, int(heads), int(kv_heads), int(head_dim), int(causal_block))
        self.items = items.to(device)
        self.lengths, self.key_lengths, self.key_starts = lengths, key_lengths, key_starts
        self.heads, self.kv_heads, self.head_dim, self.causal_block = int(heads), int(kv_heads), int(head_dim), int(causal_block)
        self.device = self.items.device


def packed_attention(q, k, v, plan, scale=None, out=None, return_lse=False):
    """softmax(scale q k^T) v for every sequence of `plan`: q [rows, heads, head_dim], k and v [key rows, kv_heads, head_dim], float16 or
    bfloat16, any strides between rows and heads.  scale > 0 (default 1 / sqrt(head_dim)).  Query head n reads key head
    n // (heads // kv_heads).

    Returns o like q, and with `return_lse` also the logarithm of each row's sum [rows, heads] (float32, not differentiable; what two results
    over different keys are joined with).  A token that sees no key: o = 0, lse = -inf, no gradient.  Rows behind the last sequence: 0 / -inf, and
    left as they were in an `out` of the caller's (no gradient through `out`, which shares no memory with q, k and v)."""
    scale = 1.0 / math.sqrt(plan.head_dim) if scale is None else float(scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        if out is not None:
            raise RuntimeError("packed_attention: out= takes no gradient; leave it out or use torch.no_grad()")
        o, lse = droid_backends.packed_attention(q, k, v, plan.items, plan.info, scale)
    else:
        o, lse, _ = droid_backends.attention_forward(q, k, v, plan.items, plan.info, scale, out)
    return (o, lse) if return_lse else o


def qk_norm_rope(q, k, positions, inv_freq, sections, q_weight=None, k_weight=None, *, normalize=True, eps=1e-6, interleaved=False, out=None):
    """q [tokens, heads, head_dim] and k [tokens, kv_heads, head_dim] (float16, bfloat16 or float32, any strides between tokens and heads),
    each head divided by the root of its mean square (+ eps) and multiplied by its weight [head_dim], then rotated by the token's position.

    positions   [tokens, axes] int32, int64 or float32: (keyframe, row, column) or fewer / more axes
    sections    pairs of channels that turn with each axis; their sum P is at most head_dim / 2, channels from 2 P on do not turn
    inv_freq    [P] float32: radians a position (positions and inv_freq get no gradient; ones that want one are refused)
    interleaved pairs are (2 i, 2 i + 1) instead of (i, P + i)
    normalize   False: rotation alone
    out         (q_out, k_out) to write to, possibly q and k themselves or rows of a cache (no gradient; they share no other memory with the
                inputs or each other)"""
    sections = [int(n) for n in sections]
    if torch.is_grad_enabled() and (positions.requires_grad or inv_freq.requires_grad):
        raise RuntimeError("qk_norm_rope: positions and inv_freq get no gradient; detach them")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        if out is not None:
            raise RuntimeError("qk_norm_rope: out= takes no gradient; leave it out or use torch.no_grad()")
        return tuple(droid_backends.qk_norm_rope(q, k, positions, inv_freq, sections, q_weight, k_weight, bool(normalize), float(eps), bool(interleaved)))
    qo, ko = out if out is not None else (None, None)
    return tuple(droid_backends.qk_norm_rope_forward(q, k, positions, inv_freq, sections, q_weight, k_weight, bool(normalize), float(eps), bool(interleaved), qo, ko))
