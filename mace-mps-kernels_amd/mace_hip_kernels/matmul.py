"""
Trainable layers on node features: ``dense``, y = act(x W^T + b) + residual with everything after the product in its
epilogue, and ``expert_dense``, the same with a weight of its own for every group of rows (elements, or experts after
``expert_order`` and ``dispatch``).  Both are differentiable in x, the weights, the bias and the residual, in float32,
bfloat16 and float16, for any number of rows from none on and any widths.

    y = dense(x, weight, bias, activation='silu', residual=x)             # x [..., K], weight [N, K], bias [N]
    h = expert_dense(rows, weights, order.offsets, biases)                # rows [R, K], weights [E, N, K], biases [E, N]

A drop-in of ``patch_model`` holds its weights as constants; these are what a model trains next to it.  The kernels are in
``csrc/mh_matmul.h``, one hipRTC module per type, product and tile; here is what chooses between them by sizes, types and
alignment, and ``csrc/mh_layers.cpp`` runs them.  A float32 product runs on the bf16 matrix cores at float32 accuracy
(operands split into three bf16 parts, six partial products; large ones as three products of float16 halves, ``halves``,
with what these do not hold computed the first way);
16-bit operands run as they are; every sum is float32 and rounded once.  The backward keeps act'(a) of the forward, not a
itself, and rounds p = g act'(a) to the type before the products that contract it.  Sums over rows that are split over
workgroups are added in a fixed order, so results are bitwise repeatable.  The reference has no such layers.
"""
import math

import torch

from . import _native, halves

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
DTYPES = {v: k for k, v in TYPES.items()}
ACTIVATIONS = {None: 0, 'relu': 1, 'silu': 2, 'gelu': 3}

# Tiles: waves (rows x columns), 16 x 16 fragments per wave (rows x columns), k per LDS buffer.  Operands of float32 and of
# unaligned 16-bit tensors pass through registers (SLOW), 16-bit ones of whole 16-byte steps go straight to LDS (FAST).
# Eight waves that share a tile rather than four measured (us): float32 64 x 64 at 1,999 x 515 x 1,021 21 / 27, at 4,096 x 1,024 x
# 1,024 61 / 72, 128 x 128 there 52 (four: 79); bfloat16 128 x 128 at 16,384 x 1,024 x 2,048 94 / 100, at 1,024 x 1,024 x 1,024
# 13.8 / 15.7, but 64 x 64 there 8.8 / 8.5.
SLOW = {
    'slow128': {4: (2, 4, 4, 2, 64), 2: (2, 4, 4, 2, 64)},
    'slow64': {4: (4, 2, 1, 2, 64), 2: (2, 2, 2, 2, 64)},
    'slow32': {4: (2, 2, 1, 1, 64)},
}
FAST = {'fast256': (2, 4, 8, 4, 64), 'fast128': (2, 4, 4, 2, 64), 'fast64': (2, 2, 2, 2, 64), 'deep64': (2, 2, 2, 2, 128)}
# What the choices between them go by, as measured: workgroups on a compute unit at once; what a round of workgroups costs
# besides the products (us, filling the first tile, storing the last); and for each product the device's rate in 1e12
# operations a second with all of those and with one each (and its own cost of a round).  In us: bfloat16 at 8,192 x 8,192 x 8,192 859 with 256 and 982 with
# 128; at 16,384 x 1,024 x 4,096 149, 163 and 234 with 256, 128 and 64; at 8,192 x 2,048 x 512 57, 27 and 28; at 600 x 2,048 x
# 1,024 22, 17.6 and 13.3 with 128, 64 and deep64, which at 16,384 x 1,024 x 2,048 takes 155 to 64's 124; unaligned at 8,001 x
# 1,023 x 2,049 87 and 106 with 128 and 64, at 4,001 x 513 x 257 15 and 10.  float32 with 128, 64 and 32: at 20,000 x 1,024 x
# 1,024 268, 314 and 400, at 20,000 x 128 x 512 32, 30 and 40, at 2,533 x 512 x 128 28, 10.9 and 9.4.
SPEED = {
    2: {'fast256': (1, 10, {'fwd': (1280, 1280), 'dx': (1280, 1280), 'dw': (1280, 1280)}),
        'fast128': (2, 4, {'fwd': (1190, 820), 'dx': (1190, 820), 'dw': (1000, 700)}),
        'fast64': (4, 3, {'fwd': (740, 320), 'dx': (740, 320), 'dw': (690, 230)}),
        'deep64': (2, 3, {'fwd': (650, 420), 'dx': (650, 420), 'dw': (650, 310)}),
        'slow128': (2, 5, {'fwd': (620, 500), 'dx': (500, 330), 'dw': (470, 320)}),
        'slow64': (4, 3, {'fwd': (380, 220), 'dx': (350, 140), 'dw': (340, 100)})},
    4: {'slow128': (1, 5, {'fwd': (181, 181), 'dx': (156, 156), 'dw': (155, 155)}),
        'slow64': (3, 3, {'fwd': (150, 125), 'dx': (140, 115), 'dw': (125, 85, 6)}),
        'slow32': (6, 2, {'fwd': (85, 38), 'dx': (85, 38), 'dw': (85, 33)}),
        'halves': (2, 5, {'fwd': (370, 300), 'dx': (370, 300), 'dw': (370, 300)})},
}
# few rows (forward): 16-row fragments, and the waves that share the contraction
FEW = {'few16': (1, 4), 'few32': (2, 4), 'few64': (4, 4)}
CUS = 256                # compute units of an MI355X
# Rows that a tile may load straight to LDS lie fewer than this many values apart: it holds their byte offsets in 31 bits
LD_MAX = 2 ** 21

_PTRS = 'const void* A, const void* B, void* C, '


def _tile(tile, dtype):
    return FAST[tile] if tile in FAST else SLOW[tile][dtype.itemsize]


def tile_shape(tile, dtype):
    """(rows, columns) of a tile."""
    if tile == 'halves':
        return halves.SIDE, halves.SIDE
    if tile in FEW:
        return 16 * FEW[tile][0], 16
    wm, wn, fm, fn = _tile(tile, dtype)[:4]
    return 16 * wm * fm, 16 * wn * fn


def tiles(dtype):
    """The tiles of a type for all three products, largest first."""
    return [*(FAST if dtype.itemsize == 2 else ()), *(t for t in SLOW if dtype.itemsize in SLOW[t])]


def symbol(mode, tile):
    """The kernel of a product's module: ``mm_fast_`` where the library is to hold operands to what FAST tiles take."""
    return f'mm_{"fast_" if tile in FAST else ""}{mode}'


def source(dtype, mode, tile=None, act=0):
    """HIP source of one module: ``mode`` 'fwd' (x W^T, with an activation), 'dx' (p W), 'dw' (p^T x), each of a ``tile``;
    'sum'."""
    ty = TYPES[dtype]
    L = [_native.layer_header('matmul')]
    if mode == 'sum':
        L += ['extern "C" __global__ __launch_bounds__(1024) void mm_sum(const float* part, void* out, const int* off, int R, '
              'int E, int L, int lg, long long n) {', f'  mm_sum_body<{ty}>(part, out, off, R, E, L, lg, n);', '}',
              'extern "C" __global__ __launch_bounds__(256) void mm_slope(const void* g, const void* slope, void* P, '
              'float* part, void* db, const int* off, long long ldg, long long ldp, int R, int N, int E, int L, int slots) {',
              f'  mm_slope_body<{ty}>(g, slope, P, part, db, off, ldg, ldp, R, N, E, L, slots);', '}']
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
    head = f'extern "C" __global__ __launch_bounds__({64 * shape[0] * shape[1]}) void {symbol(mode, tile)}({_PTRS}'
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
                m = _native.Module(code, {kind: (symbol(mode, tile), 64 * waves, *tile_shape(tile, dtype))})
        _MODULES[key] = m
    return m


def _seconds(tile, dtype, mode, tiles, depth, longest=0):
    """A product's time by SPEED: ``tiles`` workgroups of a contraction of ``depth`` on average, ``longest`` at most."""
    bm, bn = tile_shape(tile, dtype)
    at_once, ramp, rates = SPEED[dtype.itemsize][tile]
    full, alone, *own = rates[mode]
    ramp = own[0] if own else ramp
    share = tiles / CUS
    if tile != 'halves':
        share = math.ceil(share)                         # of the compute units with most
    # whole steps of 64 along k
    work, most = (2e-12 * bm * bn * 64 * math.ceil(k / 64) * CUS for k in (depth, max(depth, longest)))
    if at_once == 1:                                     # whole rounds
        return max(max(1, share) * (work / full + ramp * 1e-6), most / full)
    return max(most / alone, share * work / full) + max(1.0, share / at_once) * ramp * 1e-6


def _names(dtype, fast):
    return FAST if fast else [t for t in SLOW if dtype.itemsize in SLOW[t]]


def _tiles(tile, rows, cols, dtype, groups):
    """Workgroups of a product of rows in groups.  Groups end in part of a tile: half a tile each on average."""
    bm, bn = tile_shape(tile, dtype)
    return max(-(-rows // bm) + (groups - 1) // 2, min(groups, rows)) * -(-cols // bn)


def _rows_plan(rows, cols, depth, dtype, groups, fast, mode):
    """(seconds, tile) of the fastest tile by _seconds, and at least the time of reading the weights."""
    t, tile = min((_seconds(t, dtype, mode, _tiles(t, rows, cols, dtype, groups), depth), t) for t in _names(dtype, fast))
    return max(t, min(groups, rows) * cols * depth * dtype.itemsize / 4.5e12 + 3e-6), tile


def _choose_tile(rows, cols, depth, dtype, groups, fast, mode):
    return _rows_plan(rows, cols, depth, dtype, groups, fast, mode)[1]


def _few_tile(rows, groups, n, K, dtype, aligned):
    """The tile for few rows per group (64 at most on average), or None where a tile of rows is faster.  Measured (us, few / a
    tile) with 1, 16 and 64 rows in each group: bfloat16, one group of 4,096 x 1,024 4.2 / 7.6, 4.8 / 7.6, 8.0 / 7.8; 64 of them
    105 / 118, 161 / 125, 355 / 166; 16 of 2,546 x 773 29 / 22, 41 / 28, 97 / 38; float32, 64 of 1,024 x 1,024 54 / 56, 69 / 75,
    164 / 139."""
    per = -(-rows // groups)
    tile = next((t for t, (fragments, _) in FEW.items() if per <= 16 * fragments), None)
    if tile is None:
        return None
    # a workgroup's time on its compute unit, in us: a start, and its steps along K, dearer with more rows; sixteen columns each
    step = (0.0013 + 0.00005 * per) * (1 if aligned else 1.7) if dtype.itemsize == 2 else 0.0025 + 0.00009 * per
    share = min(groups, rows) * -(-n // 16) / CUS
    few = 3e-6 + max(1.0, share) * (0.3 + step * K) * 1e-6
    # 2 us: what staging a tile costs before the first product; in float32 _seconds is a fifth short for groups of few rows
    other = _rows_plan(rows, n, K, dtype, groups, dtype.itemsize == 2 and aligned, 'fwd')[0]
    return tile if few < other * (1.0 if dtype.itemsize == 2 else 1.2) + 2e-6 else None


def _outer_best(R, M, N, groups, grouped, dtype, fast):
    """(seconds, tile, L, slots) of a sum over R rows: whole groups (L 0), or pieces of L rows in ``slots`` slots whose parts are
    written and read once more; the fastest by _seconds and those bytes."""
    best = None
    for tile in _names(dtype, fast):
        bm, bn = tile_shape(tile, dtype)
        tiles = -(-M // bm) * -(-N // bn)
        # the longest group is what the unsplit form waits for: of few groups, taken as two and a half times the mean one
        t = _seconds(tile, dtype, 'dw', tiles * groups, R / groups, R / groups * (2.5 if 1 < groups <= 64 else 1.0))
        best = min(best or (t, tile, 0, groups), (t, tile, 0, groups))
        for pieces in (2, 4, 8, 16, 32, 64):
            L = -(-max(256, -(-R // pieces)) // 64) * 64
            if L >= R:
                break
            slots = -(-R // L) + (groups if grouped else 0)
            filled = -(-R // L) + (groups - 1) // 2
            t = _seconds(tile, dtype, 'dw', tiles * filled, L) + filled * M * N * 8 / 4.5e12 + 5e-6
            if slots <= 65535 and slots * M * N <= 2 ** 28:
                best = min(best, (t, tile, L, slots))
    return best


def _outer_plan(*args):
    return _outer_best(*args)[1:]


def _halves_pieces(R, groups, grouped, tiles):
    """(L, slots) of a weight gradient by halves: two workgroups per compute unit, each of 256 rows at least."""
    if tiles * groups >= CUS or R <= 256:
        return 0, groups
    L = max(256, -(-R // max(1, 2 * CUS // tiles)))
    L = -(-L // 64) * 64
    return L, -(-R // L) + (groups if grouped else 0)


def _by_halves(R, N, K, groups, grouped, mode):
    """Whether a float32 product goes by halves."""
    f32 = torch.float32
    if 2 * max(N, K) > LD_MAX - 64 or groups * N >= 2 ** 31:
        return False
    if mode == 'dw':
        L, slots = _halves_pieces(R, groups, grouped, -(-N // halves.SIDE) * -(-K // halves.SIDE))
        tiles = -(-N // halves.SIDE) * -(-K // halves.SIDE) * slots
        product = _seconds('halves', f32, mode, tiles, L or R / groups) + (slots * N * K * 8 / 4.5e12 if L else 0.0)
        direct = _outer_best(R, N, K, groups, grouped, f32, False)[0]
    else:
        cols, depth = (N, K) if mode == 'fwd' else (K, N)
        stored = 4 * R * cols / 4.5e12
        product = _seconds('halves', f32, mode, _tiles('halves', R, cols, f32, groups), depth) + stored
        direct = _rows_plan(R, cols, depth, f32, groups, False, mode)[0] + stored
    return halves.pays(R, N, K, groups, mode, product, direct)


def _padding_pays(slow, fast, moved, copies):
    """Whether copies of ``moved`` bytes (read and written) to whole steps of 16 bytes are worth a fast tile: ``slow`` and
    ``fast``, the seconds of the best tile of either kind."""
    return slow - fast > 1.2 * (moved / 4.5e12 + 5e-6 * copies)


def handle(m):
    """A module's handle as a number (0: none), for plans."""
    return 0 if m is None else m.handle.value


def planner(kind):
    """Makes a function ``_layers.so``'s planner of a kind.  It keeps the numbers by the arguments; ``cache_clear()`` has it ask
    again."""
    def register(fn):
        _native.PLANNERS[kind] = fn
        fn.cache_clear = lambda: _native.layers().clear_plans()
        return fn
    return register


@planner(_native.PLAN_FORWARD)
def _fwd_plan(device, dtype, R, n, K, groups, act, x_ok, w_ok, *_):
    """[module, whether by halves, modules of the halves and of the copies, whether x and the weight are copied first to whole
    steps of 16 bytes]; x_ok, w_ok: whether they come in such."""
    device, dtype = torch.device('cuda', device), DTYPES[dtype]
    if dtype == torch.float32 and R > 0 and _by_halves(R, n, K, groups, False, 'fwd'):
        return [handle(halves.module(device, 'fwd', act)), 1, handle(halves.module(device, 'split')), 0, 0, 0]
    few = _few_tile(R, groups, n, K, dtype, bool(x_ok and w_ok))
    if few:
        return [handle(module(device, dtype, 'fwd', few, act)), 0, 0, 0, 0, 0]
    fast = pad = dtype.itemsize == 2 and K <= LD_MAX - 8 and groups * n < 2 ** 31
    if fast and not (x_ok and w_ok):
        slow, quick = (_rows_plan(R, n, K, dtype, groups, q, 'fwd')[0] for q in (False, True))
        fast = pad = _padding_pays(slow, quick, 4 * K * (R * (not x_ok) + groups * n * (not w_ok)), 2 - x_ok - w_ok)
    pads = [pad and not x_ok, pad and not w_ok]
    return [handle(module(device, dtype, 'fwd', _choose_tile(R, n, K, dtype, groups, fast, 'fwd'), act)), 0, 0,
            handle(module(device, dtype, 'sum') if any(pads) else None), *map(int, pads)]


@planner(_native.PLAN_BACKWARD)
def _bwd_plan(device, dtype, R, N, K, groups, grouped, made_p, g_ok, w_ok, x_ok, need, *_):
    """[modules of the sums, of dx, of dW, of halves; rows per piece and pieces of db; of dW; floats of scratch; whether dx and
    dW go by halves; whether g, the weight and x are copied to whole steps first].  need: bits of dx, dW, db; made_p: with an
    activation, whose product g act'(a) comes in whole steps."""
    device, dtype = torch.device('cuda', device), DTYPES[dtype]
    want_x, want_w, want_b = (bool(need >> i & 1) for i in range(3))
    some = R > 0 and N > 0 and K > 0
    hx, hw = (want and some and dtype == torch.float32 and _by_halves(R, N, K, groups, grouped, mode)
              for want, mode in ((want_x, 'dx'), (want_w, 'dw')))
    # db: pieces of rows for about eight workgroups per compute unit (two / four / eight / sixteen: 100 / 100 / 69 / 73 us at
    # 16,384 x 4,096 bfloat16, 84 / 55 / 41 / 48 at 2,048 in eight groups); few rows are one piece that needs no second sum
    Ls = R if R <= 64 and not grouped else min(256, max(16, -(-R * -(-N // 256) // (8 * CUS) // 4) * 4))
    Ls = max(1, Ls)
    slots = max(1, -(-R // Ls)) + (groups if grouped else 0)
    scratch = slots * N if want_b and (grouped or slots > 1) else 0
    p_ok = made_p or g_ok
    fast_x = fast_w = dtype.itemsize == 2 and some and max(N, K) <= LD_MAX - 8 and groups * N < 2 ** 31
    if fast_x:
        if not (p_ok and w_ok):
            fast_x = want_x and _padding_pays(*(_rows_plan(R, K, N, dtype, groups, q, 'dx')[0] for q in (False, True)),
                                              4 * (R * N * (not p_ok) + groups * N * K * (not w_ok)), 2 - p_ok - w_ok)
        if not (p_ok and x_ok):
            fast_w = want_w and _padding_pays(*(_outer_best(R, N, K, groups, grouped, dtype, q)[0] for q in (False, True)),
                                              4 * R * (N * (not p_ok) + K * (not x_ok)), 2 - p_ok - x_ok)
    rows = outer = None
    if hx:
        rows = halves.module(device, 'dx')
    elif want_x and R and K:
        rows = module(device, dtype, 'dx', _choose_tile(R, K, N, dtype, groups, fast_x, 'dx'))
    Lo, slots_o = 0, groups
    if hw:
        outer = halves.module(device, 'dw')
        Lo, slots_o = _halves_pieces(R, groups, grouped, -(-N // halves.SIDE) * -(-K // halves.SIDE))
    elif want_w and N and K:
        tile, Lo, slots_o = _outer_plan(R, N, K, groups, grouped, dtype, fast_w)
        outer = module(device, dtype, 'dw', tile)
    scratch = max(scratch, slots_o * N * K if Lo else 0)
    pads = ((want_x and fast_x or want_w and fast_w) and not p_ok, want_x and fast_x and not w_ok,
            want_w and fast_w and not x_ok)
    return [handle(module(device, dtype, 'sum')), handle(rows), handle(outer),
            handle(halves.module(device, 'split') if hx or hw else None), Ls, slots, Lo, slots_o, scratch, int(hx), int(hw),
            *map(int, pads)]


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


def _check(x, weight, bias, activation, residual, lead):
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


def refused(name):
    return RuntimeError(f'mace_hip_kernels: {name} did not take its arguments')


def dense(x, weight, bias=None, activation=None, residual=None):
    """act(x weight^T + bias) + residual for x [..., K], weight [N, K], bias [N], residual [..., N], all of one type
    (float32, bfloat16 or float16) on one GPU; activation None, 'relu', 'silu' or 'gelu' (by erf).  Sums are float32, the
    result is rounded once.  Infinite and NaN values act as in a float32 sum.  x and residual may be rows of a wider
    tensor (any distance between rows); other strides are copied.  First-order backward to all four tensors (forward-mode
    tangents are refused); in the 16-bit types with an activation it rounds the gradient of x weight^T + bias to the type before
    its two products, as separate layers would: relative errors of dx and dweight are then 1.4 times one rounding's."""
    y = _native.layers().dense(x, weight, bias, residual, ACTIVATIONS.get(activation, -1), None)
    if y is None:
        _check(x, weight, bias, activation, residual, ())
        raise refused('dense')
    return y


def expert_dense(x, weight, offsets, bias=None, activation=None, residual=None):
    """``dense`` with a weight per group of rows: rows offsets[e] to offsets[e + 1] - 1 of x [R, K] take weight[e] (weight
    [E, N, K], bias [E, N], offsets [E + 1] int32 on the GPU, not decreasing, as ``expert_order`` gives them, or a part of
    these with the part's weights).  Empty groups are fine (their weights' gradients are zero); rows of no group, before the
    first or behind the last, come out as zeros and get zero gradients.  The offsets
    are not read back: contents outside [0, R] give wrong rows, no error."""
    y = None
    if torch.is_tensor(offsets):
        y = _native.layers().dense(x, weight, bias, residual, ACTIVATIONS.get(activation, -1), offsets)
    if y is None:
        _check(x, weight, bias, activation, residual, ('E',))
        if x.dim() != 2:
            raise ValueError(f'x must be rows [R, K], got {list(x.shape)}')
        E = weight.shape[0]
        if not torch.is_tensor(offsets) or offsets.dtype != torch.int32 or offsets.device != x.device:
            raise TypeError(f'offsets must be an int32 tensor on {x.device}')
        if E < 1 or tuple(offsets.shape) != (E + 1,):
            raise ValueError(f'offsets must be [{E + 1}] for {E} weights (at least one), got {list(offsets.shape)}')
        raise refused('expert_dense')
    return y
