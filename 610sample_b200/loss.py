"""Cross entropy of a linear layer (a language model's head) without keeping its logits.

    loss = linear_cross_entropy(x, weight, targets)        # mean over the rows that count

computes `F.cross_entropy(F.linear(x, weight).float(), targets)`, but the [n, V] logits exist only tile by tile: the
forward reduces each tile to a maximum and a sum per row, the backward forms the gradient of a piece of the
vocabulary at a time, in at most 512 MB (or 1024 columns), whatever V is.  Logits are summed and used in float32, never
rounded to the input type.  The reference takes the loss of whole logits (e2e/ttt_pytorch/model.py:540-671).
There is no fallback: importing this module fails if the compiled extension `attention_cuda` is missing.
"""
try:  # used as part of the package
    from . import attention_cuda as _attention_cuda
except ImportError:  # used the reference's way: this directory on sys.path
    import attention_cuda as _attention_cuda

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def linear_cross_entropy(x, weight, targets, ignore_index=-100, reduction="mean"):
    """x: (..., d); weight: (V, d), both fp16, bf16 or fp32 CUDA tensors of one type; targets: int64, (...).

    A row whose target is `ignore_index` has loss and, beside finite weights, gradients 0 and does not count in the mean; what x
    holds there, infinities and NaN too, has no influence.  A target outside [0, V) otherwise gives a NaN loss (and no fault).
    reduction: "mean" over the rows that count (NaN if none does), "sum", or "none" (the losses, shaped as targets).
    Returns float32.  Half types with d a multiple of 8 run on the tensor cores, all else on the CUDA cores.
    Twice differentiable in x and weight; the second derivative is computed by PyTorch operations, in pieces of rows."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'none', 'sum' or 'mean', got {reduction!r}")
    if x.dim() == 0 or tuple(x.shape[:-1]) != tuple(targets.shape):
        raise RuntimeError("targets must have the shape of x without its last axis")
    loss = _attention_cuda.linear_cross_entropy(x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x, weight,
                                                targets.reshape(-1) if targets.dim() != 1 else targets, ignore_index,
                                                _REDUCTIONS[reduction])
    return loss.reshape(targets.shape) if reduction == "none" and targets.dim() != 1 else loss
