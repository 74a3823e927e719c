"""Compact rows: a matrix in microscaled 8-bit ("mxfp8") or 4-bit ("mxfp4") floating point on the MI355X.

What a design matrix is in practice -- the activations that a network hands to its output layer -- carries far fewer
digits than fp64 or fp32, and the row operators of this package are bound by its bytes.  ``CompactRows`` keeps a row in
blocks of 32 columns, one scale byte (a power of two) and 32 codes each: 33 or 17 bytes where fp64 takes 256.

    X8   = compact.quantise(X)                       # E4M3
    obj  = WeightedGLMObjective(X8, y, prior=1.0)    # value, gradient, HVP and the CG route read the 8-bit rows
    hvp  = cg.GLMHessianVectorProduct(obj, theta, w)
    dW   = rows.gemm_tn(X8, dZ)                      # weight gradient of a layer with several outputs
    T    = rows.gemm_nt(compact.quantise(Q, "mxfp4"), compact.quantise(X, "mxfp4"))      # scores of all pairs

An element is off by at most 2^-4 (E4M3) or 2^-2 (E2M1) of its size, or half the smallest step of its block, whichever is
larger: a number far below the largest of its 32 reads as 0.  The smallest step is at most 2^-16 (E4M3) or 1/7 (E2M1) of the
block's largest magnitude, but never under 2^-136 (E4M3) or 2^-128 (E2M1).

The reference keeps its arrays in fp64 and has no counterpart.
"""
import torch

from . import _lib, device as dev

FORMATS = tuple(_lib.MX_FORMAT)
BLOCK = 32
_BLOCK_BYTES = {"mxfp4": 16, "mxfp8": 32}
TYPE = {torch.float64: 0, torch.float32: 1, torch.bfloat16: 2, torch.float16: 3}      # VT_TYPE_*


def check_format(format):
    if format not in FORMATS:
        raise ValueError("format must be one of %s, got %r" % (FORMATS, format))
    return format


# torch.cuda.current_stream(device).cuda_stream without the Stream object (2.8 -> 0.1 us a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_of(device):
    """The current stream of ``device`` as the C-ABI takes it."""
    if _raw_stream is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def call(name, device, run):
    """``run(stream)``, a call of the entry point ``name``, with ``device`` the current one (kernels are launched there)."""
    if device.index == torch.cuda.current_device():
        code = run(stream_of(device))
    else:
        with torch.cuda.device(device):
            code = run(stream_of(device))
    if code != _lib.VT_OK:
        _lib.check(code, name)


class CompactRows:
    """(N, D) rows in ``format``: ``codes`` (N, ceil(D / 32) * 32 or * 16 bytes) and ``scales`` (N, ceil(D / 32) bytes),
    CUDA uint8 tensors laid out as include/vittles_hip.h says.  Codes and scales made elsewhere can be handed in; the
    object holds the tensors (copied only if their layout does not suit the kernels)."""

    def __init__(self, codes, scales, D, format="mxfp8"):
        self.format = check_format(format)
        self.D = int(D)
        if self.D < 1:
            raise ValueError("D must be at least 1")
        nb = (self.D + BLOCK - 1) // BLOCK
        for name, t, width in (("codes", codes, nb * _BLOCK_BYTES[format]), ("scales", scales, nb)):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8 or t.ndim != 2 or t.shape[1] != width:
                raise ValueError("%s must be an (N, %d) uint8 tensor for %d columns in %s" % (name, width, self.D, format))
        if not (codes.is_cuda and scales.is_cuda):
            raise ValueError("codes and scales must be on the GPU")
        if codes.shape[0] != scales.shape[0] or codes.device != scales.device:
            raise ValueError("codes and scales must have the same rows and device")
        # (the kernels take row strides as they are, but rows of codes begin on 16 bytes)
        if codes.stride(1) != 1 or codes.data_ptr() % 16 or dev.ld(codes) % 16 or dev.ld(codes) < codes.shape[1]:
            codes = codes.clone(memory_format=torch.contiguous_format)
        if scales.stride(1) != 1 or dev.ld(scales) < nb:
            scales = scales.contiguous()
        self.codes, self.scales = codes, scales

    @classmethod
    def _made(cls, codes, scales, D, format):
        """The object for tensors that were made here."""
        self = cls.__new__(cls)
        self.codes, self.scales, self.D, self.format = codes, scales, D, format
        return self

    @property
    def shape(self):
        return (self.codes.shape[0], self.D)

    @property
    def device(self):
        return self.codes.device

    @property
    def dtype(self):
        """The storage type, as the objectives and row operators ask for it: the format's name."""
        return self.format

    @property
    def nbytes(self):
        return self.codes.numel() + self.scales.numel()

    def c_args(self):
        """codes, ldc, scales, lds of the C-ABI."""
        codes, scales = self.codes, self.scales
        if codes.shape[0] > 1:
            return codes.data_ptr(), codes.stride(0), scales.data_ptr(), scales.stride(0)
        return codes.data_ptr(), codes.shape[1], scales.data_ptr(), scales.shape[1]

    def c_format(self):
        return _lib.MX_FORMAT[self.format]

    def dequantise(self, dtype=torch.float32):
        """The values as an (N, D) tensor."""
        if dtype not in TYPE:
            raise TypeError("dequantise: dtype must be one of %s" % (tuple(TYPE),))
        lib = dev.require_gpu()
        device, shape = self.device, self.shape
        out = torch.empty(*shape, dtype=dtype, device=device)
        call("vt_mx_dequantise", device, lambda stream: lib.vt_mx_dequantise(
            self.c_format(), *self.c_args(), *shape, TYPE[dtype], out.data_ptr(), self.D, stream))
        return out

    def __repr__(self):
        return "CompactRows(%d x %d, %s, %s)" % (self.shape + (self.format, self.device))


def quantise(X, format="mxfp8", device=None):
    """``X`` (N, D) -- numpy, or a float64 / float32 / bfloat16 / float16 tensor -- as ``CompactRows``.

    A block's scale is the smallest power of two with which its largest magnitude still rounds to a code; codes are
    rounded to nearest, ties to even, once.  A block with a NaN, an infinity or a magnitude beyond float32 reads as NaN; a
    number that rounds to 2^128 (1.9375 2^127 and up in mxfp8, 1.75 2^127 and up in mxfp4) reads as an infinity."""
    check_format(format)
    lib = dev.require_gpu()
    if isinstance(X, torch.Tensor):
        if X.dtype not in TYPE:
            raise TypeError("quantise: X must be float64, float32, bfloat16 or float16, got %s" % X.dtype)
        if X.requires_grad:
            X = X.detach()
        if device is not None or not X.is_cuda:
            X = dev.to_device(X, device, dtype=X.dtype)
    else:
        X = dev.to_device(X, device)
    if X.ndim != 2 or X.shape[1] < 1:
        raise ValueError("X must be (N, D) with D >= 1")
    N, D = X.shape
    if N > 0 and (X.stride(1) != 1 or dev.ld(X) < D):
        X = X.contiguous()
    nb = (D + BLOCK - 1) // BLOCK
    width, at = nb * _BLOCK_BYTES[format], X.device
    codes = torch.empty(N, width, dtype=torch.uint8, device=at)      # (sizes one by one: 0.4 us less than as a tuple)
    scales = torch.empty(N, nb, dtype=torch.uint8, device=at)
    call("vt_mx_quantise", at, lambda stream: lib.vt_mx_quantise(
        TYPE[X.dtype], X.data_ptr(), dev.ld(X), N, D, _lib.MX_FORMAT[format], codes.data_ptr(), width, scales.data_ptr(), nb, stream))
    return CompactRows._made(codes, scales, D, format)
