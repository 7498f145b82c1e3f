"""
Trainable layers on node features: ``dense``, y = act(x W^T + b) + residual with everything after the product in its
epilogue, and ``expert_dense``, the same with a weight of its own for every group of rows (elements, or experts after
``expert_order`` and ``dispatch``).  Both are differentiable in x, the weights, the bias and the residual, in float32,
bfloat16 and float16, for any number of rows from none on and any widths.

    y = dense(x, weight, bias, activation='silu', residual=x)             # x [..., K], weight [N, K], bias [N]
    h = expert_dense(rows, weights, order.offsets, biases)                # rows [R, K], weights [E, N, K], biases [E, N]

A drop-in of ``patch_model`` holds its weights as constants; these are what a model trains next to it.  The kernels are in
``csrc/mh_matmul.h``, one hipRTC module per type, product and tile.  A float32 product runs on the bf16 matrix cores at
float32 accuracy (operands split into three bf16 parts, six partial products); 16-bit operands run as they are; every sum
is float32 and rounded once.  The backward keeps act'(a) of the forward, not a itself.  Sums over rows that are split over
workgroups are added in a fixed order, so results are bitwise repeatable.  The reference has no such layers.
"""
import torch

from . import _native

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {None: 0, 'relu': 1, 'silu': 2, 'gelu': 3}

# tiles: waves (rows x columns), 16 x 16 fragments per wave (rows x columns), k per LDS buffer, buffers; for float32 and the
# 16-bit types (float32 keeps three bf16 planes and two accumulators)
TILES = {
    'large': {4: (2, 2, 4, 4, 32, 1), 2: (2, 2, 4, 4, 64, 2)},
    'small': {4: (2, 2, 2, 2, 32, 1), 2: (2, 2, 2, 2, 64, 2)},
}
CUS = 256                # compute units of an MI355X

_PTRS = 'const void* A, const void* B, void* C, '


def tile_shape(tile, dtype):
    """(rows, columns) of a tile."""
    wm, wn, fm, fn, _, _ = TILES[tile][dtype.itemsize]
    return 16 * wm * fm, 16 * wn * fn


def source(dtype, mode, tile=None):
    """HIP source of one module: ``mode`` 'fwd' (x W^T), 'dx' (p W), 'dw' (p^T x), each of a ``tile``; 'sum', 'slope'."""
    ty = TYPES[dtype]
    L = [_native.layer_header('matmul')]
    if mode in ('sum', 'slope'):
        L += ['extern "C" __global__ __launch_bounds__(256) void mm_sum(const float* part, void* out, const int* off, int R, '
              'int E, int L, long long n) {', f'  mm_sum_body<{ty}>(part, out, off, R, E, L, n);', '}',
              'extern "C" __global__ __launch_bounds__(256) void mm_slope(const void* g, const void* slope, void* P, '
              'float* part, const int* off, long long ldg, int R, int N, int E, int L) {',
              f'  mm_slope_body<{ty}>(g, slope, P, part, off, ldg, R, N, E, L);', '}']
        return '\n'.join(L) + '\n'
    wm, wn, fm, fn, bk, bufs = TILES[tile][dtype.itemsize]
    shape = f'{wm}, {wn}, {fm}, {fn}, {bk}, {bufs}'
    head = f'extern "C" __global__ __launch_bounds__({64 * wm * wn}) void mm_{mode}({_PTRS}'
    if mode == 'dw':
        L += [head + 'float* part, const int* off, long long lda, long long ldb, int R, int M, int N, int E, int L) {',
              f'  mm_outer_body<{ty}, {shape}>(A, B, C, part, off, lda, ldb, R, M, N, E, L);', '}']
    else:
        L += [head + 'const void* bias, const void* res, void* slope, const int* off, long long lda, long long ldr, int R, '
              'int N, int K, int E, int act) {',
              f'  mm_rows_body<{ty}, {"true" if mode == "dx" else "false"}, {shape}>(A, B, C, bias, res, slope, off, lda, ldr, '
              'R, N, K, E, act);', '}']
    return '\n'.join(L) + '\n'


_MODULES = {}


def module(device, dtype, mode, tile=None):
    """The loaded module (compiled on first use, kept per device)."""
    key = (device.index, dtype, mode, tile)
    m = _MODULES.get(key)
    if m is None:
        code = _native.compile_source(source(dtype, mode, tile))
        with torch.cuda.device(device):
            if mode == 'sum':
                m = _native.Module(code, {_native.MH_MM_SUM: ('mm_sum', 256, 1), _native.MH_MM_SLOPE: ('mm_slope', 256, 1)})
            else:
                wm, wn = TILES[tile][dtype.itemsize][:2]
                kind = _native.MH_MM_OUTER if mode == 'dw' else _native.MH_MM_ROWS
                m = _native.Module(code, {kind: (f'mm_{mode}', 64 * wm * wn, *tile_shape(tile, dtype))})
        _MODULES[key] = m
    return m


def rows_of(t, width):
    """``t`` [..., width] as rows [R, width] whose elements are contiguous (copied only where they are not), and the
    distance between rows."""
    t = t.reshape(-1, width) if width else t.reshape(t.shape[:-1].numel(), 0)
    if t.shape[0] <= 1 or width == 0:
        return t.contiguous(), width
    if (width > 1 and t.stride(1) != 1) or t.stride(0) < width:
        t = t.contiguous()
    return t, t.stride(0)


def _choose_tile(rows, cols, dtype, groups=1):
    """The large tile where its tiles fill the compute units, else the small one."""
    bm, bn = tile_shape('large', dtype)
    return 'large' if (-(-rows // bm) + groups - 1) * -(-cols // bn) >= CUS else 'small'


def _product(x, ld, weight, bias, res, act, offsets, groups, n, keep, mode='fwd'):
    """(out [R, n], act' of it or None) of rows x [R, K]; ``mode`` 'dx': weight [.., K, n], else [.., n, K]."""
    R, K = x.shape
    out = torch.empty(R, n, device=x.device, dtype=x.dtype)
    slope = None
    if keep:
        slope = torch.empty(R, n, device=x.device, dtype=torch.float32 if x.dtype == torch.float32 else torch.uint16)
    if R and n:
        m = module(x.device, x.dtype, mode, _choose_tile(R, n, x.dtype, groups))
        P = _native.ptr
        r, ldr = (None, 0) if res is None else rows_of(res, n)
        _native.launch(f'mm_{mode}', _native.load().mh_mm_rows, m.handle, P(x), ld, P(weight), P(out), P(bias), P(r), ldr,
                       P(slope), P(offsets), R, n, K, groups, act, _native.stream_of(x))
    return out, slope


def _pieces(R, groups, per, tiles, step):
    """(L, slots) of a sum over R rows split over workgroups: about two workgroups per compute unit in all, each at
    least 256 rows; L 0 where the groups' tiles fill the device by themselves."""
    if tiles * groups >= CUS or R <= 256:
        return 0, groups
    want = max(1, 2 * CUS // tiles)
    L = max(256, -(-R // want))
    L = -(-L // step) * step
    return L, -(-R // L) + (groups if per else 0)


def _outer(p, ldp, x, ldx, offsets, groups):
    """dW [groups, M, N] = per group, sum over its rows of p^T x."""
    R, M = p.shape
    N = x.shape[1]
    dev, dt, P, lib = x.device, x.dtype, _native.ptr, _native.load()
    out = torch.empty(groups, M, N, device=dev, dtype=dt)
    if not (M and N):
        return out
    bm, bn = tile_shape('large', dt)
    tile = 'large' if -(-M // bm) * -(-N // bn) * groups >= CUS // 2 else 'small'
    bm, bn = tile_shape(tile, dt)
    L, slots = _pieces(R, groups, offsets is not None, -(-M // bm) * -(-N // bn), TILES[tile][dt.itemsize][4])
    part = torch.empty(slots, M, N, device=dev, dtype=torch.float32) if L else None
    s = _native.stream_of(x)
    _native.launch('mm_dw', lib.mh_mm_outer, module(dev, dt, 'dw', tile).handle, P(p), ldp, P(x), ldx, P(out), P(part),
                   P(offsets), R, M, N, groups, L, slots, s)
    if L:
        _native.launch('mm_sum', lib.mh_mm_sum, module(dev, dt, 'sum').handle, P(part), P(out), P(offsets), R, groups, L,
                       M * N, s)
    return out


def _slope(g, ldg, slope, offsets, groups, want_p, want_b):
    """(p = g act', sums of its columns per group), each where wanted."""
    R, N = g.shape
    dev, dt, P, lib = g.device, g.dtype, _native.ptr, _native.load()
    p = torch.empty(R, N, device=dev, dtype=dt) if want_p else None
    db = torch.empty(groups, N, device=dev, dtype=dt) if want_b else None
    # pieces of rows: about four workgroups per compute unit
    L = min(256, max(16, -(-R * -(-N // 256) // (4 * CUS) // 4) * 4))
    slots = -(-R // L) + (groups if offsets is not None else 0)
    part = torch.empty(slots, N, device=dev, dtype=torch.float32) if want_b else None
    s = _native.stream_of(g)
    m = module(dev, dt, 'sum').handle
    if R and N:
        _native.launch('mm_slope', lib.mh_mm_slope, m, P(g), ldg, P(slope), P(p), P(part), P(offsets), R, N, groups, L, slots, s)
    if want_b and N:
        _native.launch('mm_sum', lib.mh_mm_sum, m, P(part), P(db), P(offsets), R, groups, L, N, s)
    return p, db


DOUBLE_BACKWARD = ('mace_hip_kernels: double backward (create_graph=True) is not available for the trainable node layers '
                   '(dense, expert_dense, dispatch, combine, block_norm)')


class _DenseFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, res, act, offsets):
        n, K = weight.shape[-2:]
        groups = weight.shape[0] if offsets is not None else 1
        x2, ld = rows_of(x, K)
        w2 = weight.contiguous()
        need = ctx.needs_input_grad
        keep = act != 0 and any(need[:3])
        out, slope = _product(x2, ld, w2, None if bias is None else bias.contiguous(), res, act, offsets, groups, n, keep)
        ctx.save_for_backward(x if need[1] else None, weight if need[0] else None, slope, offsets)
        ctx.shapes = (x.shape, weight.shape, None if bias is None else bias.shape)
        return out.reshape(*x.shape[:-1], n)

    @staticmethod
    def backward(ctx, g):
        if torch.is_grad_enabled():          # only true under create_graph=True
            raise RuntimeError(DOUBLE_BACKWARD)
        x, weight, slope, offsets = ctx.saved_tensors
        xs, ws, bs = ctx.shapes
        n, K = ws[-2:]
        groups = ws[0] if offsets is not None else 1
        need = ctx.needs_input_grad
        dx = dw = db = None
        g2, ldg = rows_of(g, n)
        p, ldp = g2, ldg
        want_p = slope is not None and (need[0] or need[1])
        if want_p or need[2]:
            made, db = _slope(g2, ldg, slope, offsets, groups, want_p, need[2])
            if want_p:
                p, ldp = made, n
        if need[0]:
            dx = _product(p, ldp, weight.contiguous(), None, None, 0, offsets, groups, K, False, 'dx')[0].reshape(xs)
        if need[1]:
            x2, ldx = rows_of(x, K)
            dw = _outer(p, ldp, x2, ldx, offsets, groups).reshape(ws)
        return dx, dw, None if db is None else db.reshape(bs), g if need[3] else None, None, None


def check_like(name, t, x, shape=None):
    """Refuses a tensor of another type or device than x, or another shape than ``shape``."""
    if not torch.is_tensor(t) or t.dtype != x.dtype or t.device != x.device:
        raise TypeError(f'{name} must be a {x.dtype} tensor on {x.device}, got '
                        f'{(t.dtype, t.device) if torch.is_tensor(t) else type(t).__name__}')
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f'{name} must be {list(shape)}, got {list(t.shape)}')


def check_rows(name, x):
    """Refuses what the kernels do not take as rows of features."""
    if not torch.is_tensor(x) or x.dtype not in TYPES:
        raise TypeError(f'{name} must be a float32, bfloat16 or float16 tensor, got '
                        f'{x.dtype if torch.is_tensor(x) else type(x).__name__}')
    if not x.is_cuda:
        raise TypeError(f'mace_hip_kernels: {name} must be a GPU tensor, got one on {x.device}')
    if x.dim() < 1:
        raise ValueError(f'{name} must have at least one dimension')
    if x.numel() // max(1, x.shape[-1]) >= 2 ** 31 - 1024 or x.shape[-1] >= 2 ** 31 - 1024:
        raise ValueError(f'{name} is too large for one launch: {list(x.shape)}')


def _checked(x, weight, bias, activation, residual, lead):
    check_rows('x', x)
    check_like('weight', weight, x)
    if weight.dim() != 2 + len(lead) or weight.shape[-1] != x.shape[-1]:
        raise ValueError(f'weight must be [{"E, " if lead else ""}N, {x.shape[-1]}], got {list(weight.shape)}')
    n = weight.shape[-2]
    if bias is not None:
        check_like('bias', bias, x, weight.shape[:-1])
    if residual is not None:
        check_like('residual', residual, x, (*x.shape[:-1], n))
    if activation not in ACTIVATIONS:
        raise ValueError(f'activation must be one of {list(ACTIVATIONS)}, got {activation!r}')
    return ACTIVATIONS[activation]


def _run(x, weight, bias, residual, act, offsets):
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _DenseFn.apply(x, weight, bias, residual, act, offsets)
    n, K = weight.shape[-2:]
    x2, ld = rows_of(x, K)
    out, _ = _product(x2, ld, weight.contiguous(), None if bias is None else bias.contiguous(), residual, act, offsets,
                      weight.shape[0] if offsets is not None else 1, n, False)
    return out.reshape(*x.shape[:-1], n)


def dense(x, weight, bias=None, activation=None, residual=None):
    """act(x weight^T + bias) + residual for x [..., K], weight [N, K], bias [N], residual [..., N], all of one type
    (float32, bfloat16 or float16) on one GPU; activation None, 'relu', 'silu' or 'gelu' (by erf).  Sums are float32, the
    result is rounded once.  Infinite and NaN values act as in a float32 sum.  x and residual may be rows of a wider
    tensor (any distance between rows); other strides are copied.  First-order backward to all four tensors."""
    return _run(x, weight, bias, residual, _checked(x, weight, bias, activation, residual, ()), None)


def expert_dense(x, weight, offsets, bias=None, activation=None, residual=None):
    """``dense`` with a weight per group of rows: rows offsets[e] to offsets[e + 1] - 1 of x [R, K] take weight[e] (weight
    [E, N, K], bias [E, N], offsets [E + 1] int32 on the GPU, not decreasing, as ``expert_order`` gives them).  Empty groups
    are fine (their weights' gradients are zero); rows of no group come out as zeros and get zero gradients.  The offsets
    are not read back: contents outside [0, R] give wrong rows, no error."""
    act = _checked(x, weight, bias, activation, residual, ('E',))
    if x.dim() != 2:
        raise ValueError(f'x must be rows [R, K], got {list(x.shape)}')
    E = weight.shape[0]
    if not torch.is_tensor(offsets) or offsets.dtype != torch.int32 or offsets.device != x.device:
        raise TypeError(f'offsets must be an int32 tensor on {x.device}')
    if E < 1 or tuple(offsets.shape) != (E + 1,):
        raise ValueError(f'offsets must be [{E + 1}] for {E} weights (at least one), got {list(offsets.shape)}')
    return _run(x, weight, bias, residual, act, offsets.contiguous())
