"""
Rows sorted by expert and back: ``expert_order`` places every (node, expert) assignment in a stable sort by expert,
``dispatch`` copies the nodes' rows to those places, ``combine`` adds them up again with their weights.  Between the two
stands a layer with weights per expert (``expert_dense`` over ``order.offsets``).

    order = expert_order(experts, n_experts)              # experts [T, k] int32 or int64; outside [0, n_experts): dropped
    rows = dispatch(x, order)                             # [T k, C]; rows of no assignment are zero
    y = combine(rows, weights, order, residual=x)         # x[t] + sum over the kept j of weights[t, j] rows[place[t, j]]

No sizes are read back: T k rows whatever the counts, the kept ones first.  Kernels in ``csrc/mh_expert_order.h`` and
``csrc/mh_experts.h``; no atomics on results, so all of it is bitwise repeatable.  The reference has no counterpart (its models mix elements by one-hot weights).
"""
import torch

from . import _native
from .matmul import TYPES, DTYPES, planner, refused, check_like, check_rows, handle

MAX_EXPERTS = 1024


class ExpertOrder:
    """``offsets`` [E + 1], ``rows`` [T k] (flat assignment t k + j at each place, -1 behind the last), ``place`` [T, k] (-1
    where dropped), all int32 on the GPU."""

    def __init__(self, offsets, rows, place, n_experts):
        self.offsets, self.rows, self.place, self.n_experts = offsets, rows, place, n_experts


def order_source():
    return _native.layer_header('expert_order')


def source(dtype):
    ty = TYPES[dtype]
    sig = 'extern "C" __global__ __launch_bounds__(256) void '
    return _native.layer_header('matmul', 'experts') + '\n'.join([
        sig + 'ex_dispatch(const void* x, const int* place, const int* offsets, void* y, long long ldx, int T, int k, int C, '
        'int E, int lg) {', f'  ex_dispatch_body<{ty}>(x, place, offsets, y, ldx, T, k, C, E, lg);', '}',
        sig + 'ex_combine(const void* y, const float* w, const int* place, const void* res, void* out, long long ldr, int T, '
        'int k, int C, int lg) {', f'  ex_combine_body<{ty}>(y, w, place, res, out, ldr, T, k, C, lg);', '}',
        sig + 'ex_combine_bwd(const void* g, const void* y, const float* w, const int* place, const int* offsets, void* dy, '
        'float* dw, long long ldg, int T, int k, int C, int E, int lg) {',
        f'  ex_combine_bwd_body<{ty}>(g, y, w, place, offsets, dy, dw, ldg, T, k, C, E, lg);', '}']) + '\n'


_MODULES = {}


def module(device, dtype=None):
    """The loaded module of a type's rows, or (None) of the sort."""
    m = _MODULES.get((device.index, dtype))
    if m is None:
        code = _native.compile_source(order_source() if dtype is None else source(dtype))
        with torch.cuda.device(device):
            if dtype is None:
                m = _native.Module(code, {_native.MH_EXPERT_HIST: ('expert_hist', 1024, 1),
                                          _native.MH_EXPERT_PLACE: ('expert_place', 1024, 1)})
            else:
                m = _native.Module(code, {_native.MH_DISPATCH: ('ex_dispatch', 256, 1),
                                          _native.MH_COMBINE: ('ex_combine', 256, 1),
                                          _native.MH_COMBINE_BWD: ('ex_combine_bwd', 256, 1)})
        _MODULES[device.index, dtype] = m
    return m


@planner(_native.PLAN_ROUTE)
def _plan(device, dtype, C, *_):
    """[module, log2 of the lanes that share a row: one 16-byte access each, a wave at most]; the sort's for no type."""
    device = torch.device('cuda', device)
    if dtype < 0:
        return [handle(module(device)), 0]
    dtype = DTYPES[dtype]
    vectors = -(-C * dtype.itemsize // 16)
    return [handle(module(device, dtype)), min(6, max(0, (vectors - 1).bit_length()))]


def expert_order(experts, n_experts):
    """The places of assignments ``experts`` [T, k] (int32 or int64 on the GPU) in a stable sort by expert; values outside
    [0, n_experts) are dropped (a router marks what exceeds an expert's capacity with -1).  n_experts up to 1024."""
    out = _native.layers().expert_order(experts, n_experts)
    if out is None:
        if not torch.is_tensor(experts) or experts.dtype not in (torch.int32, torch.int64):
            raise TypeError('experts must be an int32 or int64 tensor')
        if not experts.is_cuda:
            raise TypeError(f'mace_hip_kernels: experts must be a GPU tensor, got one on {experts.device}')
        if experts.dim() != 2 or experts.shape[1] < 1:
            raise ValueError(f'experts must be [T, k] with k >= 1, got {list(experts.shape)}')
        if not 1 <= n_experts <= MAX_EXPERTS:
            raise ValueError(f'n_experts must be between 1 and {MAX_EXPERTS}, got {n_experts}')
        raise ValueError(f'too many assignments for one launch: {experts.numel()}')
    return ExpertOrder(*out, n_experts)


def _check_order(order, device):
    if not isinstance(order, ExpertOrder):
        raise TypeError(f'order must come from expert_order, got {type(order).__name__}')
    if order.place.device != device:
        raise TypeError(f'the order is on {order.place.device}, the rows on {device}')
    for name, t, dims in (('place', order.place, 2), ('offsets', order.offsets, 1)):
        if t.dtype != torch.int32 or t.dim() != dims or not t.is_contiguous():
            raise ValueError(f'order.{name} must be as expert_order made it (int32, {dims} dimensions, contiguous), got {t.dtype} '
                             f'{list(t.shape)}')
    if order.place.shape[1] < 1 or order.offsets.shape[0] < 2:
        raise ValueError(f'the order has no experts: place {list(order.place.shape)}, offsets {list(order.offsets.shape)}')


def dispatch(x, order):
    """The rows of x [T, C] at their places [T k, C] (x[t] at place[t, j] for every kept j); the places behind the last kept
    one are zero rows.  Backward: dx[t] = sum over the kept j of the gradient at place[t, j]."""
    y = _native.layers().dispatch(x, order.place, order.offsets) if isinstance(order, ExpertOrder) else None
    if y is None:
        check_rows('x', x)
        _check_order(order, x.device)
        if x.dim() != 2 or x.shape[0] != order.place.shape[0]:
            raise ValueError(f'x must be [{order.place.shape[0]}, C], got {list(x.shape)}')
        raise refused('dispatch')
    return y


def combine(y, weights, order, residual=None):
    """residual[t] + sum over the kept j of weights[t, j] y[place[t, j]] for rows y [T k, C] in expert order; weights [T, k]
    float32 or of y's type (None: 1), residual [T, C].  Dropped assignments are not read, whatever their weight.  A node
    without any kept one comes out as its residual (or zeros).  Backward to all three (dropped weights get 0)."""
    out = None
    if isinstance(order, ExpertOrder):
        out = _native.layers().combine(y, weights, residual, order.place, order.offsets)
    if out is None:
        check_rows('y', y)
        _check_order(order, y.device)
        T, k = order.place.shape
        if y.dim() != 2 or y.shape[0] != T * k:
            raise ValueError(f'y must be [{T * k}, C], got {list(y.shape)}')
        if weights is not None:
            if not torch.is_tensor(weights) or weights.dtype not in (torch.float32, y.dtype) or weights.device != y.device:
                raise TypeError(f'weights must be float32 or {y.dtype} on {y.device}')
            if weights.shape != (T, k):
                raise ValueError(f'weights must be [{T}, {k}], got {list(weights.shape)}')
            weights = weights.float()
        if residual is not None:
            check_like('residual', residual, y, (T, y.shape[1]))
        out = _native.layers().combine(y, weights, residual, order.place, order.offsets)
        if out is None:
            raise refused('combine')
    return out
