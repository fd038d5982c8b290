"""What a model does before and between the layers' own operators, on libwkv6_gfx950.so: the embedding and the layer norm with the residual
addition before it, with their gradients.  Not part of the reference's operator package: its model (rwkv6_model.py:187-208, :259-274) takes both from the
framework above it.

    embedding(ids, weight, scale=1.0)       rows of a table by token
    layer_norm(x, weight, bias, add=None)   the norm of x, or of the sum x + add, which is returned beside it

Tensors are bf16, fp16 or fp32 on the GPU.  A stream (x, a table) may be in fp32 while what goes beside it (add and the norm's output, the rows that are read) is in 16
bits.  All arithmetic is in fp32, and each result is rounded once.  Calls go to the current stream of the tensors' device, allocate nothing
but their results and workspaces, never synchronise, and can be captured into a graph.  Sums over tokens are always added up in the same order: the
same call gives the same bits.  The functions have first derivatives; a derivative of a gradient that was taken with create_graph is refused.
"""
import torch

from . import _native

_CODES = {torch.bfloat16: _native.BF16, torch.float16: _native.F16, torch.float32: _native.F32}
MOST_CHANNELS = 32768   # of layer_norm


def _goes_with(dtype, other):
    return other == dtype or (dtype == torch.float32 and other in _CODES)


def embedding(ids, weight, scale=1.0, padding_id=None, dtype=None):
    """scale * weight[ids]: of ids' shape and the table's width.  Differentiable in weight (V, C); its gradient is dense, and the rows that are added up
    in it need not be sorted.

    ids: int64 of any shape.  A negative id gives a row of zeros and takes no part in the gradient, an id of V or more gives a row of NaN and takes
    no part either.  padding_id: a token whose row gets no gradient.  dtype: of the result, the table's or 16 bits beside a table in fp32."""
    assert isinstance(weight, torch.Tensor) and weight.is_cuda and weight.dim() == 2 and weight.dtype in _CODES, \
        "weight must be (tokens, channels) in bfloat16, float16 or float32 on the GPU"
    assert ids.dtype == torch.int64 and ids.device == weight.device, "ids must be int64, on the table's device"
    assert weight.shape[0] > 0 and weight.shape[1] > 0, "the table is empty"
    assert padding_id is None or 0 <= padding_id < weight.shape[0], "padding_id must be a token of the table"
    dtype = weight.dtype if dtype is None else dtype
    assert _goes_with(weight.dtype, dtype), "dtype must be the table's, or 16 bits beside a table in float32"
    if ids.numel() == 0:
        return weight[:0].sum().to(dtype) * weight.new_zeros((*ids.shape, weight.shape[1]), dtype=dtype)
    return _native.load_torch().embedding(ids.contiguous(), weight, float(scale), -1 if padding_id is None else int(padding_id), _CODES[dtype])


def layer_norm(x, weight=None, bias=None, eps=1e-5, add=None, dtype=None):
    """(s - mean) / sqrt(variance + eps) * weight + bias over the last dimension (at most 32768 channels) of s = x, or of s = x + add; then returns (the norm, s).
    s has x's dtype and is rounded to it first.  Differentiable in x, add, weight and bias.

    weight, bias: (C,) of one dtype, or None.  add: of x's shape.  dtype: of the norm, x's or 16 bits beside an fp32 x (None: x's)."""
    assert isinstance(x, torch.Tensor) and x.is_cuda and x.dtype in _CODES and x.dim() >= 1, "x must be bfloat16, float16 or float32 on the GPU"
    C = x.shape[-1]
    assert 0 < C <= MOST_CHANNELS, "x must have 1 to %d channels" % MOST_CHANNELS
    for p in (weight, bias):
        assert p is None or (p.shape == (C,) and p.device == x.device and p.dtype in _CODES), "weight and bias must be (channels,), on x's device"
    assert weight is None or bias is None or weight.dtype == bias.dtype, "weight and bias must have one dtype"
    assert eps >= 0
    dtype = x.dtype if dtype is None else dtype
    assert _goes_with(x.dtype, dtype), "dtype must be x's, or 16 bits beside an x in float32"
    if add is not None:
        assert add.shape == x.shape and add.device == x.device and _goes_with(x.dtype, add.dtype), "add must be like x, in its dtype or in 16 bits beside an x in float32"
    if x.numel() == 0:
        total = x if add is None else x + add.to(x.dtype)
        y = torch.nn.functional.layer_norm(total, (C,), None if weight is None else weight.to(x.dtype), None if bias is None else bias.to(x.dtype), eps).to(dtype)
        return y if add is None else (y, total)
    branch = dtype
    if add is not None and add.dtype != dtype:
        # (the kernels take both in one type: fp32 then, and the narrower of the two is converted)
        branch, add = torch.float32, add.to(torch.float32)
    y, total = _native.load_torch().layer_norm(x, add, weight, bias, float(eps), _CODES[branch])
    if branch != dtype:
        y = y.to(dtype)
    return y if add is None else (y, total)
