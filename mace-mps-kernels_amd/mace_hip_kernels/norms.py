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
from .matmul import CUS, DOUBLE_BACKWARD, TYPES, check_like, check_rows, module as mm_module

MAX_CHANNELS = 8192


def shape(C, dtype):
    """(threads per row, vectors of 16 bytes per thread): the fewest of a wave (four rows a workgroup) or a workgroup of 128
    to 1024 threads that hold the row in one vector each, two for the longest rows of float32: the backward then keeps its
    rows and the next one's loads in registers (two vectors of 16-bit values a thread take 300)."""
    vectors = -(-C * dtype.itemsize // 16)
    tpr = next((t for t in (64, 128, 256, 512) if vectors <= t), 1024)
    return tpr, -(-vectors // tpr)


def _launch(tpr):
    """(threads, rows) of a workgroup."""
    return (256, 4) if tpr == 64 else (tpr, 1)


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


def _forward(x, y, gate, scale, wp, wn, eps, layer, gmode, keep):
    C = x.shape[-1]
    T = x.numel() // C if C else 0
    n = torch.empty_like(x)
    h = x if y is None else torch.empty_like(x)
    stats = torch.empty(T, 4, device=x.device, dtype=torch.float32) if keep else None
    if T:
        tpr, nv = shape(C, x.dtype)
        P = _native.ptr
        _native.launch('nm_fwd', _native.load().mh_norm_fwd,
                       module(x.device, x.dtype, tpr, nv, layer, y is not None, gmode).handle, P(x), P(y), P(gate), P(scale),
                       P(wp), P(wn), None if y is None else P(h), P(n), P(stats), T, C, eps, _native.stream_of(x))
    return h, n, stats


class _BlockNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, scale, wp, wn, eps, layer, gmode):
        h, n, stats = _forward(x, y, gate, scale, wp, wn, eps, layer, gmode, True)
        ctx.save_for_backward(x, y, gate, scale, wp, wn, stats)
        ctx.args = layer, gmode
        ctx.set_materialize_grads(False)
        return n if y is None else (h, n)

    @staticmethod
    def backward(ctx, *grads):
        if torch.is_grad_enabled():          # only true under create_graph=True
            raise RuntimeError(DOUBLE_BACKWARD)
        x, y, gate, scale, wp, wn, stats = ctx.saved_tensors
        layer, gmode = ctx.args
        need = ctx.needs_input_grad
        gh, gn = (None, grads[0]) if y is None else grads
        if gh is None and gn is None:
            return (None,) * 9
        gh, gn = (None if g is None else g.contiguous() for g in (gh, gn))
        C = x.shape[-1]
        T = x.numel() // C if C else 0
        dev, dt, P, lib = x.device, x.dtype, _native.ptr, _native.load()
        dx, dy, dgate = (torch.empty_like(t) if w else None for t, w in zip((x, y, gate), need[:3]))
        dsum = torch.empty((3, C), device=dev, dtype=dt) if any(need[3:6]) else None
        tpr, nv = shape(C, dt)
        blocks = _backward_blocks(T, tpr)
        part = None if dsum is None else torch.empty((blocks, 3, C), device=dev, dtype=torch.float32)
        _native.launch('nm_bwd', lib.mh_norm_bwd, module(dev, dt, tpr, nv, layer, y is not None, gmode).handle,
                       mm_module(dev, dt, 'sum').handle, P(gh), P(gn), P(x), P(y), P(gate), P(scale), P(wp), P(wn), P(stats),
                       P(dx), P(dy), P(dgate), P(part), P(dsum), T, C, blocks, _native.stream_of(x))
        return (dx, dy, dgate, *(dsum[i] if w else None for i, w in enumerate(need[3:6])), None, None, None)


def block_norm(x, y=None, gate=None, scale=None, post_weight=None, pre_weight=None, eps=1e-6, kind='rms'):
    """(h, n): h = x + scale gate norm(y) post_weight and n = norm(h) pre_weight, per row of x [..., C] (y None: h is x and
    gate, scale and post_weight must be None).  y [..., C]; gate [..., C] or [..., 1]; the weights [C], each 1 where None;
    all of one type (float32, bfloat16 or float16).  kind 'rms' or 'layer' (the mean subtracted first).  n is formed from h
    before h is rounded to the type.  C up to 8192.  First-order backward to every tensor given."""
    check_rows('x', x)
    C = x.shape[-1]
    if not 1 <= C <= MAX_CHANNELS:
        raise ValueError(f'x must have between 1 and {MAX_CHANNELS} channels, got {C}')
    if kind not in ('rms', 'layer'):
        raise ValueError(f"kind must be 'rms' or 'layer', got {kind!r}")
    if not eps >= 0:
        raise ValueError(f'eps must not be negative, got {eps}')
    gmode = 0
    if y is None:
        if gate is not None or scale is not None or post_weight is not None:
            raise ValueError('gate, scale and post_weight belong to a branch y')
    else:
        check_like('y', y, x, x.shape)
    if gate is not None:
        # [..., 1] is one value a row, also where there is one channel
        check_like('gate', gate, x)
        if gate.shape[:-1] != x.shape[:-1] or gate.dim() != x.dim() or gate.shape[-1] not in (1, C):
            raise ValueError(f'gate must be {[*x.shape[:-1], C]} or {[*x.shape[:-1], 1]}, got {list(gate.shape)}')
        gmode = 1 if gate.shape[-1] == 1 else 2
    for name, w in (('scale', scale), ('post_weight', post_weight), ('pre_weight', pre_weight)):
        if w is not None:
            check_like(name, w, x, (C,))
    ts = [None if t is None else t.contiguous() for t in (x, y, gate, scale, post_weight, pre_weight)]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        out = _BlockNormFn.apply(*ts, float(eps), kind == 'layer', gmode)
        return (x, out) if y is None else out
    h, n, _ = _forward(*ts, float(eps), kind == 'layer', gmode, False)
    return (x if y is None else h), n
