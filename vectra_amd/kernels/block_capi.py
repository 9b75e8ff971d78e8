"""ctypes binding of the block C ABI (include/vectra_block.h): what a caller
without torch.ops writes.  Tensors only supply device pointers, sizes and
strides; matrices are 2-D with unit element stride."""

import ctypes

import torch

from vectra_amd.kernels import _native

F32, F16, BF16 = 0, 1, 2
DTYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
ACTIVATIONS = {'none': 0, 'relu': 1, 'gelu': 2, 'gelu_tanh': 3, 'silu': 4}
NORMS = {'none': 0, 'rms': 1, 'layer': 2}

OK = 0
ERR_NULL_ARGUMENT = 1
ERR_BAD_DTYPE = 2
ERR_BAD_SHAPE = 3
ERR_BAD_STRUCT = 4
ERR_TOO_LARGE = 5
ERR_LAUNCH = 6
ERR_BAD_OPTION = 7
ERR_WORKSPACE = 8

# Widest row of a norm.
NORM_WIDTH = 16384

# Exported functions, as declared in include/vectra_block.h.
EXPORTS = (
    'vectra_dropout',
    'vectra_norm_forward',
    'vectra_norm_backward',
    'vectra_norm_backward_workspace_bytes',
    'vectra_blocks_quantize',
    'vectra_linear8_forward',
    'vectra_linear8_workspace_bytes',
    'vectra_block_status_string',
    'vectra_block_abi_version',
)


def _fields(*groups):
    """struct_size, then the fields of each (type, names)."""
    return [('struct_size', ctypes.c_int64)] + [(n, kind) for kind, names in groups for n in names]


_VECTORS = ('weight', 'bias', 'gate', 'post_weight', 'post_bias')
_NORM_SCALARS = (
    (ctypes.c_int32, ('dtype', 'stream_dtype') + tuple(v + '_dtype' for v in _VECTORS) + ('norm', 'post', 'threshold')),
    (ctypes.c_uint32, ('stream_id',)),
    (ctypes.c_float, ('eps', 'residual_scale')),
    (ctypes.c_int64, ('rows', 'width', 'gate_rows')),
)


class NormArgs(ctypes.Structure):
    """struct vectra_norm_args."""

    _fields_ = _fields(
        (ctypes.c_void_p, ('x', 'residual') + _VECTORS + ('rng', 'h', 'n', 'codes', 'scales')), *_NORM_SCALARS,
        (ctypes.c_int64, ('x_stride', 'residual_stride', 'gate_stride', 'h_stride', 'n_stride')))


class NormGradArgs(ctypes.Structure):
    """struct vectra_norm_grad_args."""

    _fields_ = _fields(
        (ctypes.c_void_p, ('grad_h', 'grad_n', 'x', 'residual', 'h', 'weight', 'gate', 'post_weight', 'post_bias', 'rng',
                           'dx', 'dresidual') + tuple('d' + v for v in _VECTORS)), *_NORM_SCALARS,
        (ctypes.c_int64, ('grad_h_stride', 'grad_n_stride', 'x_stride', 'residual_stride', 'h_stride', 'gate_stride',
                          'dx_stride', 'dresidual_stride', 'dgate_stride')))


class Linear8Args(ctypes.Structure):
    """struct vectra_linear8_args."""

    _fields_ = _fields(
        (ctypes.c_void_p, ('x', 'codes', 'scales', 'weight', 'weight_scales', 'bias', 'residual', 'out')),
        (ctypes.c_int32, ('dtype', 'bias_dtype', 'activation', 'gated')),
        (ctypes.c_int64, ('rows', 'width', 'width_out', 'x_stride', 'residual_stride', 'out_stride')))


class BlockError(RuntimeError):
    """A non-zero status from the block C ABI."""

    def __init__(self, status: int):
        self.status = status
        super().__init__(f'vectra block C ABI status {status}: {status_string(status)}')


def status_string(status: int) -> str:
    return _native.block_library().vectra_block_status_string(status).decode()


def abi_version() -> tuple[int, int]:
    v = _native.block_library().vectra_block_abi_version()
    return v >> 16, v & 0xFFFF


def threshold_of(p: float) -> int:
    """The t of 65536 equally likely values below which an element is dropped."""
    return round(p * 65536)


def _pointer(t):
    return None if t is None else t.data_ptr()


def _set(a, **tensors):
    for name, t in tensors.items():
        setattr(a, name, _pointer(t))
        if t is not None and hasattr(a, name + '_stride'):
            setattr(a, name + '_stride', t.stride(0))


def _norm_options(a, width_of, stream_of, vectors, gate_rows, norm, post, p, stream_id, eps, residual_scale):
    a.struct_size = ctypes.sizeof(a)
    a.rows, a.width = width_of.shape
    a.gate_rows = max(a.rows, 1) if gate_rows is None else gate_rows
    a.dtype, a.stream_dtype = DTYPES[width_of.dtype], DTYPES[stream_of.dtype]
    for name in _VECTORS:
        t = vectors.get(name)
        setattr(a, name + '_dtype', a.dtype if t is None else DTYPES[t.dtype])
    a.norm, a.post, a.threshold = NORMS[norm], NORMS[post], threshold_of(p)
    a.stream_id, a.eps, a.residual_scale = stream_id, eps, residual_scale


def make_norm_args(x, residual, *, h, n=None, codes=None, scales=None, weight=None, bias=None, gate=None,
                   post_weight=None, post_bias=None, gate_rows=None, norm='rms', post='none', p=0.0, rng=None,
                   stream_id=0, eps=1e-6, residual_scale=1.0) -> NormArgs:
    """struct vectra_norm_args of 2-D tensors; gate_rows: all rows if not given."""
    a = NormArgs()
    vectors = dict(weight=weight, bias=bias, gate=gate, post_weight=post_weight, post_bias=post_bias)
    _norm_options(a, x, residual, vectors, gate_rows, norm, post, p, stream_id, eps, residual_scale)
    _set(a, x=x, residual=residual, h=h, n=n, codes=codes, scales=scales, rng=rng, **vectors)
    return a


def make_norm_grad_args(grad_n, grad_h, *, x=None, residual=None, h=None, weight=None, gate=None, post_weight=None,
                        post_bias=None, dx=None, dresidual=None, dweight=None, dbias=None, dgate=None,
                        dpost_weight=None, dpost_bias=None, gate_rows=None, norm='rms', post='none', p=0.0, rng=None,
                        stream_id=0, eps=1e-6, residual_scale=1.0) -> NormGradArgs:
    """struct vectra_norm_grad_args of 2-D tensors: the branch's type from grad_n or x,
    the stream's from grad_h, the residual or h."""
    a = NormGradArgs()
    given = dict(weight=weight, gate=gate, post_weight=post_weight, post_bias=post_bias)
    wanted = dict(weight=dweight, bias=dbias, gate=dgate, post_weight=dpost_weight, post_bias=dpost_bias)
    vectors = {v: given.get(v) if given.get(v) is not None else wanted[v] for v in _VECTORS}
    branch = next(t for t in (grad_n, x, dx) if t is not None)
    stream = next((t for t in (grad_h, residual, h, dresidual) if t is not None), branch)
    _norm_options(a, branch, stream, vectors, gate_rows, norm, post, p, stream_id, eps, residual_scale)
    _set(a, grad_n=grad_n, grad_h=grad_h, x=x, residual=residual, h=h, rng=rng, dx=dx, dresidual=dresidual, **given,
         **{'d' + v: t for v, t in wanted.items()})
    return a


def make_linear8_args(x, weight, weight_scales, *, out, scales=None, width=None, bias=None, residual=None,
                      activation='none', gated=False) -> Linear8Args:
    """struct vectra_linear8_args of 2-D tensors; with `scales`, x holds 8-bit rows of
    `width` elements."""
    a = Linear8Args()
    a.struct_size = ctypes.sizeof(Linear8Args)
    a.rows, a.width_out = out.shape
    if scales is None:
        _set(a, x=x)
        a.width = x.shape[1]
    else:
        a.codes, a.scales = _pointer(x), _pointer(scales)
        a.width = x.shape[1] if width is None else width
    _set(a, weight=weight, weight_scales=weight_scales, bias=bias, residual=residual, out=out)
    a.dtype = DTYPES[out.dtype]
    a.bias_dtype = a.dtype if bias is None else DTYPES[bias.dtype]
    a.activation, a.gated = ACTIVATIONS[activation], int(gated)
    return a


def _run(device, stream, call, need=0, workspace=None):
    """call(workspace pointer, its size, stream) on `stream` of `device`."""
    if need < 0:
        raise BlockError(-need)
    with torch.cuda.device(device):
        own = torch.cuda.current_stream() if stream is None else torch.cuda.ExternalStream(stream)
        if workspace is None and need > 0:
            # Memory of the stream that uses it: the allocator may hand it on once
            # this call returns, but only to what that stream runs afterwards.
            with torch.cuda.stream(own):
                workspace = torch.empty(need, dtype=torch.uint8, device=device)
        status = call(_pointer(workspace), 0 if workspace is None else workspace.numel(), own.cuda_stream)
    if status != OK:
        raise BlockError(status)


def _sized(name, size, a, device, workspace, stream):
    lib = _native.block_library()
    with torch.cuda.device(device):
        need = getattr(lib, size)(ctypes.byref(a))
    _run(device, stream, lambda w, n, s: getattr(lib, name)(ctypes.byref(a), w, n, s), need, workspace)


def dropout(x, p, rng, *, out, stream_id=0, stream=None):
    """vectra_dropout into `out`, which may be x."""
    lib = _native.block_library()
    rows, width = x.shape
    _run(x.device, stream, lambda w, n, s: lib.vectra_dropout(
        _pointer(x), DTYPES[x.dtype], rows, width, x.stride(0), _pointer(out), out.stride(0), threshold_of(p),
        _pointer(rng), stream_id, s))
    return out


def norm_forward(x, residual, *, stream=None, **arguments):
    """vectra_norm_forward of make_norm_args' arguments."""
    a = make_norm_args(x, residual, **arguments)
    lib = _native.block_library()
    _run(x.device, stream, lambda w, n, s: lib.vectra_norm_forward(ctypes.byref(a), s))


def norm_backward(grad_n, grad_h, *, workspace=None, stream=None, **arguments):
    """vectra_norm_backward of make_norm_grad_args' arguments, into those gradients
    that are given."""
    a = make_norm_grad_args(grad_n, grad_h, **arguments)
    device = (grad_n if grad_n is not None else grad_h).device
    _sized('vectra_norm_backward', 'vectra_norm_backward_workspace_bytes', a, device, workspace, stream)


def quantize(x, *, codes, scales, tiles=False, stream=None):
    """vectra_blocks_quantize into `codes` and `scales`."""
    lib = _native.block_library()
    rows, width = x.shape
    _run(x.device, stream, lambda w, n, s: lib.vectra_blocks_quantize(
        _pointer(x), DTYPES[x.dtype], rows, width, x.stride(0), int(tiles), _pointer(codes), _pointer(scales), s))


def linear8(x, weight, weight_scales, *, workspace=None, stream=None, **arguments):
    """vectra_linear8_forward of make_linear8_args' arguments; returns `out`."""
    a = make_linear8_args(x, weight, weight_scales, **arguments)
    _sized('vectra_linear8_forward', 'vectra_linear8_workspace_bytes', a, x.device, workspace, stream)
    return arguments['out']
