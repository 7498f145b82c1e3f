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
import math

import torch

from . import _native, halves

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {None: 0, 'relu': 1, 'silu': 2, 'gelu': 3}

# Tiles: waves (rows x columns), 16 x 16 fragments per wave (rows x columns), k per LDS buffer.  Operands of float32 and of
# unaligned 16-bit tensors pass through registers (SLOW, also the buffers: float32 keeps three bf16 planes and two
# accumulators; two buffers, 32 k and a 128 x 128 tile of it all measured slower), 16-bit ones of whole 16-byte steps go
# straight to LDS (FAST).
SLOW = {
    'slow128': {2: (2, 2, 4, 4, 64, 2)},
    'slow64': {4: (2, 2, 2, 2, 64, 1), 2: (2, 2, 2, 2, 64, 2)},
    'slow32': {4: (2, 2, 1, 1, 64, 1)},
}
FAST = {'fast256': (2, 4, 8, 4, 64), 'fast128': (2, 2, 4, 4, 64), 'fast64': (2, 2, 2, 2, 64)}
# What the choices between them go by, as measured: workgroups on a compute unit at once, the device's rate in 1e12
# operations a second with all of those and with one each, and what a round of workgroups costs besides (us, filling the first
# tile, storing the last).  bfloat16 at 8,192 x 8,192 x 8,192 859 us with 256 and 982 with 128; at 16,384 x 1,024 x 4,096 149,
# 163 and 234 with 256, 128 and 64; at 8,192 x 2,048 x 512 58, 27 and 28; at 1,024 x 1,024 x 1,024 32, 15 and 11.  float32 with
# 64 and 32: at 20,000 x 128 x 512 36 and 46, at 2,533 x 512 x 128 21 and 13, at 700 x 1,000 x 900 30 and 23.
SPEED = {
    2: {'fast256': (1, 1280, 1280, 10), 'fast128': (2, 1120, 780, 5), 'fast64': (4, 740, 350, 3),
        'slow128': (2, 800, 480, 5), 'slow64': (4, 620, 300, 3)},
    4: {'slow64': (3, 150, 70, 3), 'slow32': (6, 110, 38, 2)},
}
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
    return [*(FAST if dtype.itemsize == 2 else ()), *(t for t in SLOW if dtype.itemsize in SLOW[t])]


def source(dtype, mode, tile=None, act=0):
    """HIP source of one module: ``mode`` 'fwd' (x W^T, with an activation), 'dx' (p W), 'dw' (p^T x), each of a ``tile``;
    'sum'."""
    ty = TYPES[dtype]
    L = [_native.layer_header('matmul')]
    if mode == 'sum':
        L += ['extern "C" __global__ __launch_bounds__(1024) void mm_sum(const float* part, void* out, const int* off, int R, '
              'int E, int L, int lg, long long n) {', f'  mm_sum_body<{ty}>(part, out, off, R, E, L, lg, n);', '}',
              'extern "C" __global__ __launch_bounds__(256) void mm_slope(const void* g, const void* slope, void* P, '
              'float* part, void* db, const int* off, long long ldg, long long ldp, int R, int N, int E, int L) {',
              f'  mm_slope_body<{ty}>(g, slope, P, part, db, off, ldg, ldp, R, N, E, L);', '}']
        if dtype.itemsize == 2:
            L += ['extern "C" __global__ __launch_bounds__(256) void mm_pad(const void* x, void* y, long long ld, int R, int K, '
                  'int Kp) {', f'  mm_pad_body<{ty}>(x, y, ld, R, K, Kp);', '}']
        return '\n'.join(L) + '\n'
    args = 'A, B, C, bias, res, slope, off, lda, ldb, ldr, R, N, K, E'
    tail = ('const void* bias, const void* res, void* slope, const int* off, long long lda, long long ldb, long long ldr, '
            'int R, int N, int K, int E) {')
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
                kinds = {_native.MH_MM_SUM: ('mm_sum', 1024, 1), _native.MH_MM_SLOPE: ('mm_slope', 256, 1)}
                if dtype.itemsize == 2:
                    kinds[_native.MH_MM_PAD] = ('mm_pad', 256, 1)
                m = _native.Module(code, kinds)
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


def _aligned(t, ld, width):
    """Whether rows of a 16-bit tensor are whole steps of 16 bytes, with a tile's offsets within 2^31 bytes."""
    return width % 8 == 0 and ld % 8 == 0 and t.data_ptr() % 16 == 0 and ld < 2 ** 21


def _up8(n):
    return -(-n // 8) * 8


def _seconds(tile, dtype, tiles, depth, longest=0):
    """A product's time by SPEED: ``tiles`` workgroups of a contraction of ``depth`` on average, ``longest`` at most."""
    bm, bn = tile_shape(tile, dtype)
    at_once, full, alone, ramp = SPEED[dtype.itemsize][tile]
    share = tiles / CUS
    work, most = (2e-12 * bm * bn * k * CUS for k in (depth, max(depth, longest)))
    if at_once == 1:                                     # whole rounds
        return max(max(1, math.ceil(share)) * (work / full + ramp * 1e-6), most / full)
    return max(most / alone, share * work / full) + max(1.0, share / at_once) * ramp * 1e-6


def _choose_tile(rows, cols, depth, dtype, groups, fast):
    """The tile that is fastest by _seconds.  Groups end in part of a tile: half a tile each on average."""
    def tiles(tile):
        bm, bn = tile_shape(tile, dtype)
        return (-(-rows // bm) + (min(groups, rows) - 1) // 2) * -(-cols // bn)
    names = FAST if fast else [t for t in SLOW if dtype.itemsize in SLOW[t]]
    return min(names, key=lambda t: _seconds(t, dtype, tiles(t), depth))


def _few_tile(rows, groups):
    """The tile for few rows per group, or None."""
    per = -(-rows // groups)
    return next((t for t, (fragments, _) in FEW.items() if per <= 16 * fragments), None)


def _outer_plan(R, M, N, groups, grouped, dtype, fast):
    """(tile, L, slots) of a sum over R rows: whole groups (L 0), or pieces of L rows in ``slots`` slots whose parts are
    written and read once more; the fastest by _seconds and those bytes."""
    best = None
    for tile in FAST if fast else [t for t in SLOW if dtype.itemsize in SLOW[t]]:
        bm, bn = tile_shape(tile, dtype)
        tiles = -(-M // bm) * -(-N // bn)
        # the longest group is what the unsplit form waits for: of few groups, taken as two and a half times the mean one
        t = _seconds(tile, dtype, tiles * groups, R / groups, R / groups * (2.5 if 1 < groups <= 64 else 1.0))
        best = min(best or (t, tile, 0, groups), (t, tile, 0, groups))
        for pieces in (2, 4, 8, 16, 32, 64):
            L = -(-max(256, -(-R // pieces)) // 64) * 64
            if L >= R:
                break
            slots = -(-R // L) + (groups if grouped else 0)
            filled = -(-R // L) + (groups - 1) // 2
            t = _seconds(tile, dtype, tiles * filled, L) + filled * M * N * 8 / 4.5e12 + 5e-6
            if slots <= 65535 and slots * M * N <= 2 ** 28:
                best = min(best, (t, tile, L, slots))
    return best[1:]


def _halves_pieces(R, groups, grouped, tiles):
    """(L, slots) of a weight gradient by halves: two workgroups per compute unit, each of 256 rows at least."""
    if tiles * groups >= CUS or R <= 256:
        return 0, groups
    L = max(256, -(-R // max(1, 2 * CUS // tiles)))
    L = -(-L // 64) * 64
    return L, -(-R // L) + (groups if grouped else 0)


def _padding_pays(flops, slow, moved, copies):
    """Whether copies of ``moved`` bytes (read and written) to whole steps of 16 bytes are worth a fast tile, for a product
    that runs at ``slow`` 1e12 operations a second through registers (forward about 600, dx 470, dW 240) and at 850 else."""
    return flops * (1 / slow - 1 / 850) * 1e-12 > 1.2 * (moved / 4.5e12 + 5e-6 * copies)


def _pad(t, ld, rows, width):
    """(rows copied to whole steps of 16 bytes with zeros behind them, their distance)."""
    to = _up8(width)
    y = torch.empty((rows, to), device=t.device, dtype=t.dtype)
    _native.launch('mm_pad', _native.load().mh_mm_pad, module(t.device, t.dtype, 'sum').handle, t.data_ptr(), ld, y.data_ptr(),
                   rows, width, to, _native.stream_of(t))
    return y, to


# What a call's sizes lead to, kept by the sizes: modules are looked up and shapes chosen once per size, not per call.
@functools.lru_cache(maxsize=4096)
def _fwd_plan(device, dtype, R, n, K, groups, act, x_ok, w_ok):
    """(module, None: by halves; whether x and the weight are copied first)."""
    if dtype == torch.float32 and halves.pays(R, n, K, groups, 'fwd'):
        return None, False, False
    few = _few_tile(R, groups)
    if few:
        return module(device, dtype, 'fwd', few, act), False, False
    fast = pad = dtype.itemsize == 2
    if fast and not (x_ok and w_ok):
        fast = pad = _padding_pays(2.0 * R * n * K, 600, 4 * K * (R * (not x_ok) + groups * n * (not w_ok)),
                                   2 - x_ok - w_ok)
    return (module(device, dtype, 'fwd', _choose_tile(R, n, K, dtype, groups, fast), act), pad and not x_ok,
            pad and not w_ok)


@functools.lru_cache(maxsize=4096)
def _bwd_plan(device, dtype, R, N, K, groups, grouped, made_p, g_ok, w_ok, x_ok, want_x, want_w, want_b):
    """(modules of the sums, of dx and of dW; rows per piece and pieces of db; of dW; floats of scratch; whether dx and dW go
    by halves; whether g, the weight and x are copied to whole steps first)."""
    some = R > 0 and N > 0 and K > 0
    hx, hw = (want and some and dtype == torch.float32 and halves.pays(R, N, K, groups, mode)
              for want, mode in ((want_x, 'dx'), (want_w, 'dw')))
    # db: pieces of rows for about eight workgroups per compute unit (two / four / eight / sixteen: 100 / 100 / 69 / 73 us at
    # 16,384 x 4,096 bfloat16, 84 / 55 / 41 / 48 at 2,048 in eight groups); few rows are one piece that needs no second sum
    Ls = R if R <= 64 and not grouped else min(256, max(16, -(-R * -(-N // 256) // (8 * CUS) // 4) * 4))
    Ls = max(1, Ls)
    slots = max(1, -(-R // Ls)) + (groups if grouped else 0)
    scratch = slots * N if want_b and (grouped or slots > 1) else 0
    p_ok = made_p or g_ok
    fast_x = fast_w = dtype.itemsize == 2 and some
    if fast_x:
        flops = 2.0 * R * N * K
        if not (p_ok and w_ok):
            fast_x = want_x and _padding_pays(flops, 470, 4 * (R * N * (not p_ok) + groups * N * K * (not w_ok)),
                                              2 - p_ok - w_ok)
        if not (p_ok and x_ok):
            fast_w = want_w and _padding_pays(flops, 240, 4 * R * (N * (not p_ok) + K * (not x_ok)), 2 - p_ok - x_ok)
    rows = outer = None
    if want_x and R and K and not hx:
        rows = module(device, dtype, 'dx', _choose_tile(R, K, N, dtype, groups, fast_x))
    Lo, slots_o = 0, groups
    if hw:
        Lo, slots_o = _halves_pieces(R, groups, grouped, -(-N // halves.SIDE) * -(-K // halves.SIDE))
    elif want_w and N and K:
        tile, Lo, slots_o = _outer_plan(R, N, K, groups, grouped, dtype, fast_w)
        outer = module(device, dtype, 'dw', tile)
    scratch = max(scratch, slots_o * N * K if Lo else 0)
    pads = ((want_x and fast_x or want_w and fast_w) and not p_ok, want_x and fast_x and not w_ok,
            want_w and fast_w and not x_ok)
    return module(device, dtype, 'sum'), rows, outer, Ls, slots, Lo, slots_o, scratch, hx, hw, pads


def _product(x, ld, weight, bias, res, act, offsets, groups, keep):
    """(out [R, n], act' of it or None) of rows x [R, K] and weight [.., n, K]."""
    R, K = x.shape
    n = weight.shape[-2]
    dev, dt = x.device, x.dtype
    out = torch.empty((R, n), device=dev, dtype=dt)
    slope = torch.empty((R, n), device=dev, dtype=torch.float32 if dt == torch.float32 else torch.uint16) if keep else None
    if R and n:
        m, pad_x, pad_w = _fwd_plan(dev, dt, R, n, K, groups, act, _aligned(x, ld, K), _aligned(weight, K, K))
        P = _native.ptr
        r, ldr = (None, 0) if res is None else rows_of(res, n)
        if m is None:
            halves.product(x, ld, weight, bias, r, ldr, act, slope, offsets, groups, out)
            return out, slope
        ldw = K
        if pad_x:
            x, ld = _pad(x, ld, R, K)
        if pad_w:
            weight, ldw = _pad(weight, K, groups * n, K)
        _native.launch('mm_fwd', _native.load().mh_mm_rows, m.handle, P(x), ld, P(weight), max(1, ldw), P(out), P(bias), P(r),
                       ldr, P(slope), P(offsets), R, n, K, groups, _native.stream_of(x))
    return out, slope


def _backward(g, ldg, slope, weight, x, ldx, offsets, groups, need):
    """(dx, dW, db) of g [R, N], each where ``need`` says so (weight or x None where what they are for is not)."""
    R, N = g.shape
    K = (x if weight is None else weight).shape[-1] if weight is not None or x is not None else 0
    want_x, want_w, want_b = need
    dev, dt, P = g.device, g.dtype, _native.ptr
    made = slope is not None
    sums, rows, outer, Ls, slots, Lo, slots_o, scratch, hx, hw, (pad_g, pad_w, pad_x) = _bwd_plan(
        dev, dt, R, N, K, groups, offsets is not None, made, made or _aligned(g, ldg, N),
        weight is not None and _aligned(weight, K, K), x is not None and _aligned(x, ldx, K), want_x, want_w, want_b)
    p, ldp, ldw = None, 0, max(1, K)
    if made:
        ldp = _up8(N) if dt != torch.float32 else N
        p = torch.empty((R, ldp), device=dev, dtype=dt)
    elif pad_g:
        g, ldg = _pad(g, ldg, R, N)
    if pad_w:
        weight, ldw = _pad(weight, K, groups * N, K)
    if pad_x:
        x, ldx = _pad(x, ldx, R, K)
    dx = torch.empty((R, K), device=dev, dtype=dt) if want_x else None
    dw = torch.empty((groups, N, K), device=dev, dtype=dt) if want_w else None
    db = torch.empty((groups, N), device=dev, dtype=dt) if want_b else None
    part = torch.empty(scratch, device=dev, dtype=torch.float32) if scratch else None
    if made or want_b or rows is not None or outer is not None:
        _native.launch('mm_bwd', _native.load().mh_mm_bwd, sums.handle, None if rows is None else rows.handle,
                       None if outer is None else outer.handle, P(g), ldg, P(slope), P(weight), ldw, P(x), ldx, P(offsets),
                       P(p), ldp, P(dx) if rows is not None else None, P(dw) if outer is not None else None, P(db), P(part), R,
                       N, K, groups, Ls, slots, Lo, slots_o, _native.stream_of(g))
    if hx or hw:
        if made:
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
