"""ctypes binding of the dense C ABI (include/vectra_dense.h): what a caller
without torch.ops writes.  Tensors only supply device pointers, sizes and
strides; matrices are 2-D with unit element stride."""

import ctypes

import torch

from vectra_amd.kernels import _native

F32, F16, BF16 = 0, 1, 2
DTYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
ACTIVATIONS = {'none': 0, 'relu': 1, 'gelu': 2, 'gelu_tanh': 3, 'silu': 4}

OK = 0
ERR_NULL_ARGUMENT = 1
ERR_BAD_DTYPE = 2
ERR_BAD_SHAPE = 3
ERR_BAD_STRUCT = 4
ERR_TOO_LARGE = 5
ERR_LAUNCH = 6
ERR_BAD_ACTIVATION = 7
ERR_WORKSPACE = 8

# Exported functions, as declared in include/vectra_dense.h.
EXPORTS = (
    'vectra_dense_forward',
    'vectra_dense_forward_workspace_bytes',
    'vectra_dense_backward',
    'vectra_dense_backward_workspace_bytes',
    'vectra_rows_quantize',
    'vectra_rows_dequantize',
    'vectra_dense_status_string',
    'vectra_dense_abi_version',
)


def _fields(pointers, ints, longs):
    return ([('struct_size', ctypes.c_int64)] + [(n, ctypes.c_void_p) for n in pointers]
            + [(n, ctypes.c_int32) for n in ints] + [(n, ctypes.c_int64) for n in longs])


class DenseArgs(ctypes.Structure):
    """struct vectra_dense_args."""

    _fields_ = _fields(
        ('x', 'weight', 'bias', 'residual', 'out'),
        ('dtype', 'bias_dtype', 'activation', 'gated'),
        ('rows', 'width_in', 'width_out', 'x_stride', 'weight_stride', 'residual_stride', 'out_stride'))


class DenseGradArgs(ctypes.Structure):
    """struct vectra_dense_grad_args."""

    _fields_ = _fields(
        ('x', 'codes', 'scales', 'weight', 'bias', 'grad', 'dx', 'dweight', 'dbias'),
        ('dtype', 'bias_dtype', 'activation', 'gated'),
        ('rows', 'width_in', 'width_out', 'x_stride', 'codes_stride', 'scales_stride', 'weight_stride',
         'grad_stride', 'dx_stride', 'dweight_stride'))


class DenseError(RuntimeError):
    """A non-zero status from the dense C ABI."""

    def __init__(self, status: int):
        self.status = status
        super().__init__(f'vectra dense C ABI status {status}: {status_string(status)}')


def status_string(status: int) -> str:
    return _native.dense_library().vectra_dense_status_string(status).decode()


def abi_version() -> tuple[int, int]:
    v = _native.dense_library().vectra_dense_abi_version()
    return v >> 16, v & 0xFFFF


def _pointer(t):
    return None if t is None else t.data_ptr()


def make_args(x, weight, bias, residual, out, activation='none', gated=False) -> DenseArgs:
    """struct vectra_dense_args of 2-D tensors."""
    a = DenseArgs()
    a.struct_size = ctypes.sizeof(DenseArgs)
    a.x, a.weight, a.bias, a.residual, a.out = map(_pointer, (x, weight, bias, residual, out))
    a.dtype = DTYPES[x.dtype]
    a.bias_dtype = a.dtype if bias is None else DTYPES[bias.dtype]
    a.activation, a.gated = ACTIVATIONS[activation], int(gated)
    a.rows, a.width_in = x.shape
    a.width_out = out.shape[1]
    a.x_stride, a.weight_stride, a.out_stride = x.stride(0), weight.stride(0), out.stride(0)
    a.residual_stride = 0 if residual is None else residual.stride(0)
    return a


def make_grad_args(grad, x, weight, bias, dx, dweight, dbias, activation='none', gated=False,
                   scales=None) -> DenseGradArgs:
    """struct vectra_dense_grad_args of 2-D tensors; with `scales`, x holds codes."""
    a = DenseGradArgs()
    a.struct_size = ctypes.sizeof(DenseGradArgs)
    if scales is None:
        a.x, a.x_stride = _pointer(x), x.stride(0)
    else:
        a.codes, a.codes_stride = _pointer(x), x.stride(0)
        a.scales, a.scales_stride = _pointer(scales), scales.stride(0)
    a.weight, a.bias, a.grad = map(_pointer, (weight, bias, grad))
    a.dx, a.dweight, a.dbias = map(_pointer, (dx, dweight, dbias))
    a.dtype = DTYPES[weight.dtype]
    given = bias if bias is not None else dbias
    a.bias_dtype = a.dtype if given is None else DTYPES[given.dtype]
    a.activation, a.gated = ACTIVATIONS[activation], int(gated)
    a.rows, a.width_in = x.shape
    a.width_out = grad.shape[1]
    a.weight_stride, a.grad_stride = weight.stride(0), grad.stride(0)
    a.dx_stride = 0 if dx is None else dx.stride(0)
    a.dweight_stride = 0 if dweight is None else dweight.stride(0)
    return a


def _call(name, a, device, workspace, stream):
    lib = _native.dense_library()
    with torch.cuda.device(device):
        need = getattr(lib, name + '_workspace_bytes')(ctypes.byref(a))
        if need < 0:
            raise DenseError(-need)
        own = torch.cuda.current_stream() if stream is None else torch.cuda.ExternalStream(stream)
        if workspace is None and need > 0:
            # Memory of the stream that uses it: the allocator may hand it on once
            # this call returns, but only to what that stream runs afterwards.
            with torch.cuda.stream(own):
                workspace = torch.empty(need, dtype=torch.uint8, device=device)
        status = getattr(lib, name)(ctypes.byref(a), _pointer(workspace),
                                    0 if workspace is None else workspace.numel(), own.cuda_stream)
    if status != OK:
        raise DenseError(status)


def forward(x, weight, bias=None, residual=None, *, out, activation='none', gated=False, workspace=None, stream=None):
    """vectra_dense_forward into `out`."""
    _call('vectra_dense_forward', make_args(x, weight, bias, residual, out, activation, gated), x.device, workspace,
          stream)
    return out


def backward(grad, x, weight, bias=None, *, dx=None, dweight=None, dbias=None, activation='none', gated=False,
             scales=None, workspace=None, stream=None):
    """vectra_dense_backward into those of dx, dweight and dbias that are given."""
    a = make_grad_args(grad, x, weight, bias, dx, dweight, dbias, activation, gated, scales)
    _call('vectra_dense_backward', a, grad.device, workspace, stream)
