"""Packed batches: sequences of different lengths laid end to end on one axis of rows, without padding.

    plan = packed_plan(cu_seqlens, n_tok)                  # once per batch, shared by all layers
    q, k = packed_qk_norm_rope(q, k, q_weight, k_weight, freqs, positions)
    O = packed_attention(q, k, v, plan)                    # [n_tok, heads, D]

Attention is causal within each sequence, optionally within a sliding window, with grouped heads: `q` has a
multiple of the heads of `k` and `v`, head h of `q` reading head h // (heads of q / heads of k).  It is
differentiable to second order, as `flash_attention_v7`; the second derivative runs on sequences of like lengths, padded to the
longest of them, in memory that goes with the batch's rows.  There is no counterpart in the reference, whose batches are dense [B, H, N, D]
(e2e/ttt_pytorch/model.py:174-191).  `packed_qk_norm_rope` is the step in front of it, as `qk_norm_rope` is
for dense batches, with positions given per token.  There is no fallback: importing this module fails if the compiled
extension `attention_cuda` is missing.
"""
import torch

try:  # used as part of the package
    from . import attention_cuda as _attention_cuda
except ImportError:  # used the reference's way: this directory on sys.path
    import attention_cuda as _attention_cuda


class PackedPlan:
    """What the kernels need to know about a batch's sequences; made by `packed_plan`."""

    __slots__ = ("tensor", "n_tok", "n_seq", "max_seqlen")

    def __init__(self, tensor, n_tok, n_seq, max_seqlen):
        self.tensor, self.n_tok, self.n_seq, self.max_seqlen = tensor, n_tok, n_seq, max_seqlen


def packed_plan(cu_seqlens, n_tok, max_seqlen=None):
    """The plan of a batch of `n_tok` rows whose sequence i is rows [cu_seqlens[i], cu_seqlens[i + 1]).

    cu_seqlens: int32 or int64 CUDA tensor of n_seq + 1 offsets, from small to large; one outside [0, n_tok] or
    below an earlier one is cut to it.  Sequences may be empty, and rows may belong to none.  The offsets are read
    on the device, by one launch on the current stream: nothing waits for the host, and a plan made inside a
    captured graph is made anew by each replay.  A later change of `cu_seqlens` does not change the plan.
    max_seqlen: length of the longest sequence, or an upper bound, if the caller knows it; only the second
    derivative uses it, which else reads the lengths from the device.  With it every sequence costs as much there as one of
    that length, and where one is longer all of the second derivative is NaN.  0 says that none is needed: it is 0."""
    if max_seqlen is not None and max_seqlen < 0:
        raise ValueError("max_seqlen must be >= 0")
    return PackedPlan(_attention_cuda.packed_plan(cu_seqlens, n_tok), n_tok, cu_seqlens.numel() - 1, max_seqlen)


def packed_attention(q, k, v, plan, window_size=None):
    """q: (n_tok, H, D); k, v: (n_tok, H_kv, D), H a multiple of H_kv; fp16, bf16 or fp32 CUDA tensors, D a
    multiple of 16 up to 128; for fp16 and bf16 views such as slices of one projection's result are read in place.

    Key j is visible to query i of the same sequence when j <= i and, with a `window_size`, i < j + window_size.
    The softmax scale is 1 / sqrt(D).  Rows that see no key (of no sequence, or a window of 0) give 0.  What
    rows of other sequences or of none hold, infinities and NaN too, has no influence on a sequence's result;
    within a sequence, an infinite or NaN row of k or v (or, in the backward, of q or the gradient) may reach rows that it is
    masked for as well, up to 255 before the first or behind the last one that it is not.
    Returns O: (n_tok, H, D), dense."""
    return _attention_cuda.packed_attention(q, k, v, plan.tensor, plan.n_tok, plan.n_seq, window_size, plan.max_seqlen)


def packed_qk_norm_rope(q, k, q_weight, k_weight, freqs, positions, sections=None, eps=1e-6):
    """RMS norm of every row of q: (n_tok, H, D) and k: (n_tok, H_kv, D) over D, times a weight, then rotation of its pairs
    (elements 2i and 2i + 1) by the angle of the token's position; one pass over both.  Returns (q, k), dense.

    q_weight, k_weight: (D,), of the type of q and k or float32; None: no norm, only the rotation.
    freqs: `qk_prep.rope_table(...)`, float32 (rows, D / 2, 2); positions: (n_tok,) or (axes, n_tok), int32 or int64, rows of
    freqs; one outside of it gives NaN, and a gradient of 0 where the result's is 0.  sections: how many of the D / 2 pairs turn with each axis, in order (up to four
    axes: time, height and width of a video's patches, say); None for positions of one axis.
    q and k may be slices of one projection's result.  D even, up to 128; fp16, bf16 or fp32.  Computed in float32 and
    rounded once (`qk_norm_rope` rounds where the reference's separate operations do).  Twice differentiable in q, k and the
    weights; the second derivative is computed by PyTorch operations."""
    if sections is None:
        if positions.dim() != 1:
            raise ValueError("positions of several axes need sections")
        sections = (q.shape[-1] // 2,)
    return tuple(_attention_cuda.packed_qk_norm_rope(q, k, q_weight, k_weight, freqs, positions, list(sections), eps))
