"""What a decoder layer does between its attention calls: layer norm, linear layers with what follows them, gated
feed-forward blocks.

    h = layer_norm(x, weight, bias)
    y = linear(h, w1, b1, activation="gelu")
    x = linear(y, w2, residual=x)
    x = gated_feed_forward(h, w_gate, w_up, w_down, residual=x)

All are differentiable to second order, as `flash_attention_v7`, with kernels for both backward passes; a third derivative is
refused.  fp16, bf16 or fp32 CUDA tensors; leading axes are rows.  The reference's model has linear layers and gated blocks as
separate eager operations (e2e/ttt_pytorch/model.py); its norms are RMS norms, where `layer_norm` is what a pre-norm decoder with
layer norm needs.  Autocast changes nothing here: no tensor is cast, so half-precision rows beside float32 weights are refused, and
float32 rows are computed in float32.  There is no fallback: importing this module fails if the compiled extension
`attention_cuda` is missing.
"""
try:  # used as part of the package
    from . import attention_cuda as _attention_cuda
except ImportError:  # used the reference's way: this directory on sys.path
    import attention_cuda as _attention_cuda

_ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "gelu_tanh": 3}


def _activation(name):
    if name not in _ACTIVATIONS:
        raise ValueError(f"activation must be None, 'silu', 'gelu' or 'gelu_tanh', got {name!r}")
    return _ACTIVATIONS[name]


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """x: (..., d), d up to 32768; weight, bias: (d,), of the type of x or both float32, either may be None.

    (x - mean) / sqrt(variance + eps) * weight + bias over the last axis, in float32, rounded once to the type of x.  Rows may be
    any distance apart.  The gradients of weight and bias have their type and are the same in every run."""
    return _attention_cuda.layer_norm(x, weight, bias, eps)


def linear(x, weight, bias=None, activation=None, residual=None):
    """activation(x weight^T + bias) + residual.  x: (..., k); weight: (m, k); bias: (m,); residual: (..., m); of one type.

    activation: None, "silu", "gelu" (with the normal distribution) or "gelu_tanh".  Sums are float32, and the result is rounded once.
    With an activation the backward keeps its argument, of half types in fp16 within its range.  Half types run on the tensor cores: slices whose rows start
    at multiples of 16 bytes are read in place, others (odd widths, transposed weights) are copied first.  float32 runs on the
    CUDA cores, without TF32."""
    return _attention_cuda.linear(x, weight, bias, residual, _activation(activation))


def gated_feed_forward(x, w_gate, w_up, w_down, activation="silu", residual=None):
    """(activation(x w_gate^T) * (x w_up^T)) w_down^T + residual.  x: (..., d); w_gate, w_up: (f, d); w_down: (m, f);
    residual: (..., m); of one type.

    Both projections, the activation and the product are one kernel, the second projection with the residual another.  The inner
    values are rounded to the type of x before the second projection; the backward keeps them and both projections, of half types
    with four bits more than 16 each: fp16 with 13 bits of mantissa up to 2^46, beyond which gradients are NaN."""
    return _attention_cuda.gated_feed_forward(x, w_gate, w_up, w_down, residual, _activation(activation))
