"""Rows in microscaled 4-bit floating point ("mx4"; include/ipx.h, ipx_mx4_quantize).

32 consecutive elements of a row share a power-of-two scale, an element is one of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} times it:
17 bytes per 32 elements. `quantize` gives the two arrays a service stores or ships (codes uint8 [n, nb, 16], scales uint8
[n, nb], nb = ceil(d / 32)); FlatIPIndex(d, storage="mx4") takes them with add_mx4, or quantises rows itself in add.
No counterpart in the reference.
"""
import ctypes as C

import numpy as np

from . import _lib

BLOCK = 32


def n_blocks(d):
    return -(-int(d) // BLOCK)


_torch = None
_raw_stream = None


def _is_torch(x):
    return type(x).__module__.startswith("torch") and hasattr(x, "data_ptr")


def torch_types():
    """{torch dtype: IPX dtype} of rows and values."""
    global _torch
    if _torch is None:
        import torch
        _torch = {torch.float32: _lib.IPX_F32, torch.float16: _lib.IPX_F16, torch.bfloat16: _lib.IPX_BF16}
    return _torch


def stream_of(device):
    """The raw handle of the current stream of a torch CUDA device."""
    global _raw_stream
    if _raw_stream is None:
        import torch
        # the raw handle costs 0.1 us, a Stream object to read it from 2 us
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
            (lambda index: torch.cuda.current_stream(index).cuda_stream)
    return _raw_stream(device.index)


def check_torch_pair(codes, scales, d, device=None):
    """(codes, scales) of n rows of d elements as CUDA tensors: shapes, types, one device. Returns them contiguous."""
    import torch
    nb, n = n_blocks(d), len(codes)
    assert codes.dtype == torch.uint8 and scales.dtype == torch.uint8
    assert codes.shape == (n, nb, 16) and scales.shape == (n, nb)
    assert codes.is_cuda and scales.device == codes.device
    assert device is None or codes.device.index == device
    return codes.contiguous(), scales.contiguous()


def check_numpy_pair(codes, scales, d):
    codes, scales = np.ascontiguousarray(codes), np.ascontiguousarray(scales)
    nb = n_blocks(d)
    assert codes.dtype == np.uint8 and scales.dtype == np.uint8
    assert codes.ndim == 3 and codes.shape[1:] == (nb, 16) and scales.shape == (codes.shape[0], nb)
    return codes, scales


def quantize(x, device=0):
    """x [n, d] -> (codes uint8 [n, nb, 16], scales uint8 [n, nb]). torch CUDA tensors (float32 / float16 / bfloat16; rows
    may be a strided view with adjacent elements) give CUDA tensors on their device, stream-ordered; numpy arrays (float32 /
    float16, anything else is converted to float32) give numpy arrays, computed on GPU `device`."""
    L = _lib.lib()
    if _is_torch(x):
        import torch
        n, d = x.shape
        dt = torch_types()[x.dtype]
        assert x.is_cuda
        if d > 1 and x.stride(1) != 1 or n > 1 and x.stride(0) < d:
            x = x.contiguous()
        nb, device = n_blocks(d), x.device
        codes = torch.empty((n, nb, 16), dtype=torch.uint8, device=device)
        scales = torch.empty((n, nb), dtype=torch.uint8, device=device)
        stride = x.stride(0) if n > 1 else d
        _lib.check(L.ipx_mx4_quantize(x.data_ptr(), n, d, stride, dt, codes.data_ptr(), scales.data_ptr(), 1, device.index,
                                      stream_of(device)))
        return codes, scales
    n, d = x.shape
    x = np.ascontiguousarray(x, dtype=x.dtype if x.dtype in (np.float32, np.float16) else np.float32)
    codes = np.empty((n, n_blocks(d), 16), dtype=np.uint8)
    scales = np.empty((n, n_blocks(d)), dtype=np.uint8)
    dt = _lib.IPX_F32 if x.dtype == np.float32 else _lib.IPX_F16
    _lib.check(L.ipx_mx4_quantize(C.c_void_p(x.ctypes.data), n, d, d, dt, C.c_void_p(codes.ctypes.data),
                                  C.c_void_p(scales.ctypes.data), 0, int(device), None))
    return codes, scales


def dequantize(codes, scales, d, dtype=None, device=0):
    """The values [n, d] that (codes, scales) stand for, as float32 unless `dtype` says otherwise (torch: float32, float16,
    bfloat16; numpy: float32, float16). Exact in float32 and bfloat16."""
    L = _lib.lib()
    d = int(d)
    if _is_torch(codes):
        import torch
        dtype = dtype or torch.float32
        dt = torch_types()[dtype]
        codes, scales = check_torch_pair(codes, scales, d)
        n, device = codes.shape[0], codes.device
        out = torch.empty((n, d), dtype=dtype, device=device)
        _lib.check(L.ipx_mx4_dequantize(codes.data_ptr(), scales.data_ptr(), n, d, out.data_ptr(), dt, 1, device.index,
                                        stream_of(device)))
        return out
    dtype = np.dtype(dtype or np.float32)
    dt = {np.dtype("float32"): _lib.IPX_F32, np.dtype("float16"): _lib.IPX_F16}[dtype]
    codes, scales = check_numpy_pair(codes, scales, d)
    out = np.empty((codes.shape[0], d), dtype=dtype)
    _lib.check(L.ipx_mx4_dequantize(C.c_void_p(codes.ctypes.data), C.c_void_p(scales.ctypes.data), codes.shape[0], d,
                                    C.c_void_p(out.ctypes.data), dt, 0, int(device), None))
    return out
