"""
``block_norm``: the norms before and after a block of layers, fused with the block's gate and residual scale.  A node's
stream x, the output y of a block on it, and the norm in front of the next block:

    u = norm(y) post_weight,   h = x + scale gate u,   n = norm(h) pre_weight                    (per row of C channels)

in one pass over x and y: h, n = block_norm(x, y, gate, scale, post_weight, pre_weight).  Without y (the first block):
h = x.  norm is v / sqrt(mean v^2 + eps) ('rms') or (v - mean v) / sqrt(var v + eps) ('layer').  The backward reads each
tensor once and gives the gradients of all of them; its sums over rows are added in a fixed order.  Kernels in
``csrc/mh_norms.h``; all sums are float32.  The reference has no counterpart.
"""
import torch

from . import _native
from .matmul import CUS, TYPES, DTYPES, planner, refused, check_like, check_rows, handle, module as mm_module

MAX_CHANNELS = 8192
KINDS = {'rms': 0, 'layer': 1}


def shape(C, dtype):
    """(threads per row, vectors of 16 bytes per thread): the fewest of a part of a wave (256 / 4 to 256 / 64 rows a workgroup)
    or a workgroup of 128 to 1024 threads that hold the row in one vector each, two for the longest rows of float32: the
    backward then keeps its rows and the next one's loads in registers (two vectors of 16-bit values a thread take 300).
    With at least a wave to a row, 32,768 rows of 64 bfloat16 values took 19.4 us forward and 42
    backward, so 6.2 and 14.4."""
    vectors = -(-C * dtype.itemsize // 16)
    tpr = next((t for t in (4, 8, 16, 32, 64, 128, 256, 512) if vectors <= t), 1024)
    return tpr, -(-vectors // tpr)


def _launch(tpr):
    """(threads, rows) of a workgroup."""
    return (256, 256 // tpr) if tpr <= 64 else (tpr, 1)


def _backward_blocks(T, tpr):
    """Workgroups of the backward: two per compute unit for each 256 threads' worth of a row (measured at 32,768 rows, us, for
    1 / 2 / 4 per compute unit: 2,048 channels bfloat16 264 / 212 / 231, 1,024 of them 158 / 128 / 176, 512 91 / 61 / 70, 1,024
    of float32 224 / 215 / 226), one for each compute unit at least (4,096 of float32, 8,000 rows, 128 / 256 workgroups:
    233 / 163), and no more than leave each row group four rows, whose sums cost as much as reading two."""
    threads, rows = _launch(tpr)
    return max(1, min(-(-T // (4 * rows)), max(CUS, 2 * CUS * 256 // threads)))


def source(dtype, tpr, nv, layer, branch, gate):
    b = lambda v: 'true' if v else 'false'  # noqa: E731
    args = f'{TYPES[dtype]}, {tpr}, {nv}, {b(layer)}, {b(branch)}, {gate}'
    sig = f'extern "C" __global__ __launch_bounds__({_launch(tpr)[0]}) void '
    return _native.layer_header('matmul', 'norms') + '\n'.join([
        sig + 'nm_fwd(const void* x, const void* y, const void* gate, const void* scale, const void* wp, const void* wn, '
        'void* h, void* n, float* stats, int T, int C, float eps) {',
        f'  nm_fwd_body<{args}>(x, y, gate, scale, wp, wn, h, n, stats, T, C, eps);', '}',
        sig + 'nm_bwd(const void* gh, const void* gn, const void* x, const void* y, const void* gate, const void* scale, '
        'const void* wp, const void* wn, const float* stats, void* dx, void* dy, void* dgate, float* part, int T, int C) {',
        f'  nm_bwd_body<{args}>(gh, gn, x, y, gate, scale, wp, wn, stats, dx, dy, dgate, part, T, C);', '}']) + '\n'


_MODULES = {}


def module(device, dtype, tpr, nv, layer, branch, gate):
    key = (device.index, dtype, tpr, nv, layer, branch, gate)
    m = _MODULES.get(key)
    if m is None:
        code = _native.compile_source(source(dtype, tpr, nv, layer, branch, gate))
        with torch.cuda.device(device):
            m = _native.Module(code, {_native.MH_NORM_FWD: ('nm_fwd', *_launch(tpr)),
                                      _native.MH_NORM_BWD: ('nm_bwd', *_launch(tpr))})
        _MODULES[key] = m
    return m


@planner(_native.PLAN_NORM)
def _plan(device, dtype, T, C, layer, branch, gate, *_):
    """[module, module of the sums, workgroups of the backward]."""
    device, dtype = torch.device('cuda', device), DTYPES[dtype]
    tpr, nv = shape(C, dtype)
    return [handle(module(device, dtype, tpr, nv, bool(layer), bool(branch), gate)), handle(mm_module(device, dtype, 'sum')),
            _backward_blocks(T, tpr)]


def _check(x, y, gate, scale, post_weight, pre_weight, eps, kind):
    check_rows('x', x)
    C = x.shape[-1]
    if not 1 <= C <= MAX_CHANNELS:
        raise ValueError(f'x must have between 1 and {MAX_CHANNELS} channels, got {C}')
    if kind not in ('rms', 'layer'):
        raise ValueError(f"kind must be 'rms' or 'layer', got {kind!r}")
    if not eps >= 0:
        raise ValueError(f'eps must not be negative, got {eps}')
    if y is None:
        if gate is not None or scale is not None or post_weight is not None:
            raise ValueError('gate, scale and post_weight belong to a branch y')
    else:
        check_like('y', y, x, x.shape)
    if gate is not None:
        check_like('gate', gate, x)
        if gate.shape[:-1] != x.shape[:-1] or gate.dim() != x.dim() or gate.shape[-1] not in (1, C):
            raise ValueError(f'gate must be {[*x.shape[:-1], C]} or {[*x.shape[:-1], 1]}, got {list(gate.shape)}')
    for name, w in (('scale', scale), ('post_weight', post_weight), ('pre_weight', pre_weight)):
        if w is not None:
            check_like(name, w, x, (C,))


def block_norm(x, y=None, gate=None, scale=None, post_weight=None, pre_weight=None, eps=1e-6, kind='rms'):
    """(h, n): h = x + scale gate norm(y) post_weight and n = norm(h) pre_weight, per row of x [..., C] (y None: h is x and
    gate, scale and post_weight must be None).  y [..., C]; gate [..., C] or [..., 1]; the weights [C], each 1 where None;
    all of one type (float32, bfloat16 or float16).  kind 'rms' or 'layer' (the mean subtracted first).  n is formed from h
    before h is rounded to the type.  C up to 8192.  First-order backward to every tensor given."""
    out = _native.layers().block_norm(x, y, gate, scale, post_weight, pre_weight, eps, KINDS.get(kind, -1))
    if out is None:
        _check(x, y, gate, scale, post_weight, pre_weight, eps, kind)
        raise refused('block_norm')
    return out
