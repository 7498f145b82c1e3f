"""
Trainable layers on node features: ``dense``, y = act(x W^T + b) + residual with everything after the product in its
epilogue, and ``expert_dense``, the same with a weight of its own for every group of rows (elements, or experts after
``expert_order`` and ``dispatch``).  Both are differentiable in x, the weights, the bias and the residual, in float32,
bfloat16 and float16, for any number of rows from none on and any widths.

    y = dense(x, weight, bias, activation='silu', residual=x)             # x [..., K], weight [N, K], bias [N]
    h = expert_dense(rows, weights, order.offsets, biases)                # rows [R, K], weights [E, N, K], biases [E, N]

A drop-in of ``patch_model`` holds its weights as constants; these are what a model trains next to it.  The kernels are in
``csrc/mh_matmul.h``, one hipRTC module per type, product and tile.  A float32 product runs on the bf16 matrix cores at
float32 accuracy (operands split into three bf16 parts, six partial products; large ones as three products of float16
halves, ``halves``); 16-bit operands run as they are; every sum is float32 and rounded once.  The backward keeps act'(a) of the forward, not a itself.  Sums over rows that are split over
workgroups are added in a fixed order, so results are bitwise repeatable.  The reference has no such layers.
"""
import functools

import torch

from . import _native, halves

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {None: 0, 'relu': 1, 'silu': 2, 'gelu': 3}

# Tiles: waves (rows x columns), 16 x 16 fragments per wave (rows x columns).  Operands of float32 and of unaligned 16-bit
# tensors pass through registers (SLOW, also k per LDS buffer and buffers: float32 keeps three bf16 planes and two
# accumulators); aligned 16-bit ones go straight to LDS (FAST).
SLOW = {
    'slow128': {4: (2, 2, 4, 4, 32, 1), 2: (2, 2, 4, 4, 64, 2)},
    'slow64': {4: (2, 2, 2, 2, 32, 1), 2: (2, 2, 2, 2, 64, 2)},
}
FAST = {'fast256': (2, 4, 8, 4, 64), 'fast128': (2, 2, 4, 4, 64), 'fast64': (2, 2, 2, 2, 64)}
# few rows (forward): 16-row fragments, and the waves that share the contraction
FEW = {'few16': (1, 4), 'few32': (2, 4), 'few64': (4, 4)}
CUS = 256                # compute units of an MI355X

_PTRS = 'const void* A, const void* B, void* C, '


def _tile(tile, dtype):
    return FAST[tile] if tile in FAST else SLOW[tile][dtype.itemsize]


def tile_shape(tile, dtype):
    """(rows, columns) of a tile."""
    if tile in FEW:
        return 16 * FEW[tile][0], 16
    wm, wn, fm, fn = _tile(tile, dtype)[:4]
    return 16 * wm * fm, 16 * wn * fn


def tiles(dtype):
    """The tiles of a type for all three products, largest first."""
    return [*(FAST if dtype.itemsize == 2 else ()), *SLOW]


def source(dtype, mode, tile=None, act=0):
    """HIP source of one module: ``mode`` 'fwd' (x W^T, with an activation), 'dx' (p W), 'dw' (p^T x), each of a ``tile``;
    'sum'."""
    ty = TYPES[dtype]
    L = [_native.layer_header('matmul')]
    if mode == 'sum':
        L += ['extern "C" __global__ __launch_bounds__(1024) void mm_sum(const float* part, void* out, const int* off, int R, '
              'int E, int L, int lg, long long n) {', f'  mm_sum_body<{ty}>(part, out, off, R, E, L, lg, n);', '}',
              'extern "C" __global__ __launch_bounds__(256) void mm_slope(const void* g, const void* slope, void* P, '
              'float* part, void* db, const int* off, long long ldg, int R, int N, int E, int L) {',
              f'  mm_slope_body<{ty}>(g, slope, P, part, db, off, ldg, R, N, E, L);', '}']
        return '\n'.join(L) + '\n'
    args = 'A, B, C, bias, res, slope, off, lda, ldr, R, N, K, E'
    tail = ('const void* bias, const void* res, void* slope, const int* off, long long lda, long long ldr, int R, int N, '
            'int K, int E) {')
    if tile in FEW:
        tm, waves = FEW[tile]
        L += [f'extern "C" __global__ __launch_bounds__({64 * waves}) void mm_{mode}({_PTRS}{tail}',
              f'  mm_few_body<{ty}, {act}, {tm}, {waves}>({args});', '}']
        return '\n'.join(L) + '\n'
    shape = _tile(tile, dtype)
    b = lambda v: 'true' if v else 'false'  # noqa: E731
    L += [f'typedef mm_{"fast_" if tile in FAST else ""}tile<{ty}, {b(mode == "dw")}, {b(mode != "fwd")}, '
          f'{", ".join(map(str, shape))}> tile_t;']
    head = f'extern "C" __global__ __launch_bounds__({64 * shape[0] * shape[1]}) void mm_{mode}({_PTRS}'
    if mode == 'dw':
        L += [head + 'float* part, const int* off, long long lda, long long ldb, int R, int M, int N, int E, int L) {',
              f'  mm_outer_body<{ty}, tile_t>(A, B, C, part, off, lda, ldb, R, M, N, E, L);', '}']
    else:
        L += [head + tail, f'  mm_rows_body<{ty}, {b(mode == "dx")}, {act}, tile_t>({args});', '}']
    return '\n'.join(L) + '\n'


_MODULES = {}


def module(device, dtype, mode, tile=None, act=0):
    """The loaded module (compiled on first use, kept per device)."""
    key = (device.index, dtype, mode, tile, act)
    m = _MODULES.get(key)
    if m is None:
        code = _native.compile_source(source(dtype, mode, tile, act))
        with torch.cuda.device(device):
            if mode == 'sum':
                m = _native.Module(code, {_native.MH_MM_SUM: ('mm_sum', 1024, 1), _native.MH_MM_SLOPE: ('mm_slope', 256, 1)})
            else:
                waves = FEW[tile][1] if tile in FEW else _tile(tile, dtype)[0] * _tile(tile, dtype)[1]
                kind = _native.MH_MM_OUTER if mode == 'dw' else _native.MH_MM_ROWS
                m = _native.Module(code, {kind: (f'mm_{mode}', 64 * waves, *tile_shape(tile, dtype))})
        _MODULES[key] = m
    return m


def rows_of(t, width):
    """``t`` [..., width] as rows [R, width] whose elements are contiguous (copied only where they are not), and the
    distance between rows."""
    if t.dim() != 2:
        t = t.reshape(-1, width) if width else t.reshape(t.shape[:-1].numel(), 0)
    if t.shape[0] <= 1 or width == 0:
        return t.contiguous(), width
    if (width > 1 and t.stride(1) != 1) or t.stride(0) < width:
        t = t.contiguous()
    return t, t.stride(0)


def _aligned(t, ld):
    """Whether the rows of a 16-bit tensor start at multiples of 16 bytes, with a tile's offsets within 2^31 bytes."""
    return ld % 8 == 0 and t.data_ptr() % 16 == 0 and ld < 2 ** 21


def _choose_tile(rows, cols, dtype, groups, fast):
    """The largest tile of which there are enough to give every compute unit one, else the smallest."""
    names = list(FAST) if fast else list(SLOW)
    for tile in names[:-1]:
        bm, bn = tile_shape(tile, dtype)
        if (-(-rows // bm) + groups - 1) * -(-cols // bn) >= CUS:
            return tile
    return names[-1]


def _few_tile(rows, groups):
    """The tile for few rows per group, or None."""
    per = -(-rows // groups)
    return next((t for t, (fragments, _) in FEW.items() if per <= 16 * fragments), None)


def _outer_tile(M, N, dtype, fast):
    """The largest tile that both sides of a weight fill: splits over rows make up for few tiles."""
    names = list(FAST) if fast else list(SLOW)
    return next((t for t in names if min(M, N) >= tile_shape(t, dtype)[0]), names[-1])


def _pieces(R, groups, per, tiles, step):
    """(L, slots) of a sum over R rows split over workgroups: about two workgroups per compute unit in all, each at
    least 256 rows; L 0 where the groups' tiles fill the device by themselves."""
    if tiles * groups >= CUS or R <= 256:
        return 0, groups
    want = max(1, 2 * CUS // tiles)
    L = max(256, -(-R // want))
    L = -(-L // step) * step
    return L, -(-R // L) + (groups if per else 0)


# What a call's sizes lead to, kept by the sizes: modules are looked up and shapes chosen once per size, not per call.
@functools.lru_cache(maxsize=4096)
def _rows_plan(device, dtype, mode, R, n, K, groups, act, aligned):
    """The module of a product over rows; None: by halves."""
    if dtype == torch.float32 and mode == 'fwd' and halves.pays(R, n, K, groups, mode):
        return None
    fast = dtype.itemsize == 2 and aligned and K % 8 == 0 and (mode == 'fwd' or n % 8 == 0)
    tile = (_few_tile(R, groups) if mode == 'fwd' else None) or _choose_tile(R, n, dtype, groups, fast)
    return module(device, dtype, mode, tile, act)


@functools.lru_cache(maxsize=4096)
def _bwd_plan(device, dtype, R, N, K, groups, grouped, g_aligned, w_aligned, x_aligned, want_x, want_w, want_b):
    """(modules of the sums, of dx and of dW; rows per piece and pieces of db; of dW; floats of scratch; whether dx and dW go
    by halves)."""
    hx, hw = (want and dtype == torch.float32 and R > 0 and N > 0 and K > 0 and halves.pays(R, N, K, groups, mode)
              for want, mode in ((want_x, 'dx'), (want_w, 'dw')))
    want_x = want_x and not hx
    rows = _rows_plan(device, dtype, 'dx', R, K, N, groups, 0, g_aligned and w_aligned) if want_x and R and K else None
    # db: pieces of rows for about eight workgroups per compute unit (two / four / eight / sixteen: 100 / 100 / 69 / 73 us at
    # 16,384 x 4,096 bfloat16, 84 / 55 / 41 / 48 at 2,048 in eight groups); few rows are one piece that needs no second sum
    Ls = R if R <= 64 and not grouped else min(256, max(16, -(-R * -(-N // 256) // (8 * CUS) // 4) * 4))
    Ls = max(1, Ls)
    slots = max(1, -(-R // Ls)) + (groups if grouped else 0)
    scratch = slots * N if want_b and (grouped or slots > 1) else 0
    outer, Lo, slots_o = None, 0, groups
    if hw:
        Lo, slots_o = _pieces(R, groups, grouped, -(-N // halves.SIDE) * -(-K // halves.SIDE), 64)
        scratch = max(scratch, slots_o * N * K if Lo else 0)
    elif want_w and N and K:
        tile = _outer_tile(N, K, dtype, dtype.itemsize == 2 and g_aligned and x_aligned and N % 8 == 0 and K % 8 == 0)
        outer = module(device, dtype, 'dw', tile)
        bm, bn = tile_shape(tile, dtype)
        Lo, slots_o = _pieces(R, groups, grouped, -(-N // bm) * -(-K // bn), 64)
        scratch = max(scratch, slots_o * N * K if Lo else 0)
    return module(device, dtype, 'sum'), rows, outer, Ls, slots, Lo, slots_o, scratch, hx, hw


def _product(x, ld, weight, bias, res, act, offsets, groups, keep):
    """(out [R, n], act' of it or None) of rows x [R, K] and weight [.., n, K]."""
    R, K = x.shape
    n = weight.shape[-2]
    dev, dt = x.device, x.dtype
    out = torch.empty((R, n), device=dev, dtype=dt)
    slope = torch.empty((R, n), device=dev, dtype=torch.float32 if dt == torch.float32 else torch.uint16) if keep else None
    if R and n:
        m = _rows_plan(dev, dt, 'fwd', R, n, K, groups, act, _aligned(x, ld) and weight.data_ptr() % 16 == 0)
        P = _native.ptr
        r, ldr = (None, 0) if res is None else rows_of(res, n)
        if m is None:
            halves.product(x, ld, weight, bias, r, ldr, act, slope, offsets, groups, out)
            return out, slope
        _native.launch('mm_fwd', _native.load().mh_mm_rows, m.handle, P(x), ld, P(weight), P(out), P(bias), P(r), ldr,
                       P(slope), P(offsets), R, n, K, groups, _native.stream_of(x))
    return out, slope


def _backward(g, ldg, slope, weight, x, ldx, offsets, groups, need):
    """(dx, dW, db) of g [R, N], each where ``need`` says so (weight or x NULL where what they are for is not)."""
    R, N = g.shape
    K = (x if weight is None else weight).shape[-1] if weight is not None or x is not None else 0
    want_x, want_w, want_b = need
    dev, dt, P = g.device, g.dtype, _native.ptr
    if slope is not None and not (want_x or want_w):
        want_p = want_b                                  # db alone still needs the product
    else:
        want_p = slope is not None
    g_aligned = want_p or _aligned(g, ldg)
    sums, rows, outer, Ls, slots, Lo, slots_o, scratch, hx, hw = _bwd_plan(
        dev, dt, R, N, K, groups, offsets is not None, N % 8 == 0 if want_p else g_aligned,
        weight is not None and weight.data_ptr() % 16 == 0, x is not None and _aligned(x, ldx), want_x, want_w, want_b)
    p = torch.empty((R, N), device=dev, dtype=dt) if want_p else None
    dx = torch.empty((R, K), device=dev, dtype=dt) if want_x else None
    dw = torch.empty((groups, N, K), device=dev, dtype=dt) if want_w else None
    db = torch.empty((groups, N), device=dev, dtype=dt) if want_b else None
    part = torch.empty(scratch, device=dev, dtype=torch.float32) if scratch else None
    if want_p or want_b or rows is not None or outer is not None:
        _native.launch('mm_bwd', _native.load().mh_mm_bwd, sums.handle, None if rows is None else rows.handle,
                   None if outer is None else outer.handle, P(g), ldg, P(slope) if want_p else None, P(weight), P(x), ldx,
                   P(offsets), P(p), P(dx) if rows is not None else None, P(dw) if outer is not None else None, P(db), P(part),
                   R, N, K, groups, Ls, slots, Lo, slots_o, _native.stream_of(g))
    if hx or hw:
        if want_p:
            g, ldg = p, N
        if hx:
            halves.input_gradient(g, ldg, weight, offsets, groups, dx)
        if hw:
            halves.weight_gradient(g, ldg, x, ldx, offsets, groups, dw, part, Lo, slots_o)
            if Lo:
                _native.launch('mm_sum', _native.load().mh_mm_sum, sums.handle, P(part), P(dw), P(offsets), R, groups, Lo,
                               N * K, _native.stream_of(g))
    return dx, dw, db


DOUBLE_BACKWARD = ('mace_hip_kernels: double backward (create_graph=True) is not available for the trainable node layers '
                   '(dense, expert_dense, dispatch, combine, block_norm)')


class _DenseFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, res, act, offsets):
        need = ctx.needs_input_grad
        K = weight.shape[-1]
        groups = weight.shape[0] if offsets is not None else 1
        x2, ld = rows_of(x, K)
        weight = weight.contiguous()
        out, slope = _product(x2, ld, weight, None if bias is None else bias.contiguous(), res, act, offsets, groups,
                              act != 0 and (need[0] or need[1] or need[2]))
        ctx.save_for_backward(x if need[1] else None, weight if need[0] else None, slope, offsets)
        ctx.sizes = x.shape, weight.shape, None if bias is None else bias.shape
        return out if x.dim() == 2 else out.view(*x.shape[:-1], out.shape[1])

    @staticmethod
    def backward(ctx, g):
        if torch.is_grad_enabled():          # only true under create_graph=True
            raise RuntimeError(DOUBLE_BACKWARD)
        x, weight, slope, offsets = ctx.saved_tensors
        xs, ws, bs = ctx.sizes
        need = ctx.needs_input_grad
        dx = dw = db = None
        if need[0] or need[1] or need[2]:
            g2, ldg = rows_of(g, ws[-2])
            x2, ldx = (None, 0) if x is None else rows_of(x, ws[-1])
            dx, dw, db = _backward(g2, ldg, slope, weight, x2, ldx, offsets, ws[0] if offsets is not None else 1, need[:3])
            dx = None if dx is None else dx.view(xs)
            dw = None if dw is None else dw.view(ws)
            db = None if db is None else db.view(bs)
        return dx, dw, db, g if need[3] else None, None, None


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
    x2, ld = rows_of(x, weight.shape[-1])
    out, _ = _product(x2, ld, weight.contiguous(), None if bias is None else bias.contiguous(), residual, act, offsets,
                      weight.shape[0] if offsets is not None else 1, False)
    return out if x.dim() == 2 else out.view(*x.shape[:-1], out.shape[1])


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
