"""
The trainable node layers where their inputs are out of the ordinary: groups that begin behind the first row, operands
that a tile cannot take, forward-mode derivatives, units far in an activation's tail, products of very unlike
magnitudes, more groups or columns than a grid dimension holds,
orders made by hand, inputs given other data before the backward.
Tolerances as in the layers' other tests, derived beside each.
"""
import numpy as np
import pytest
import torch

import mace_hip_kernels as mhk
from mace_hip_kernels import _native, halves, matmul
from test_node_layers_gpu import ACTS, BF16, E32, F16, F32, TINY, U, by_halves, dense_case, dev, near, rand  # noqa: F401

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize('dt', [F32, BF16, F16], ids=['f32', 'bf16', 'f16'])


def poison(*shapes, dt):
    """Leaves NaN in the memory that the next tensors of these shapes get."""
    for _ in range(3):
        kept = [torch.full(s, float('nan'), dtype=dt, device='cuda') for s in shapes for _ in range(3)]
        del kept


# ------------------------------------------------------------------------------------------ rows before the first group
def _behind_leading_rows(dt, lead=290):
    """expert_dense over offsets that begin at ``lead``: rows before the first group and behind the last are zero, with zero
    gradients, and the groups are as ever."""
    d = dev()
    rng = np.random.default_rng(lead)
    R, K, N = lead + 410, 64, 72
    off = [lead, lead, lead + 210, lead + 350]
    x, w, b, g = rand(rng, R, K, dt=dt), rand(rng, 3, N, K, dt=dt, scale=K ** -0.5), rand(rng, 3, N, dt=dt), rand(rng, R, N, dt=dt)
    res = rand(rng, R, N, dt=dt)
    for rows in (slice(0, lead), slice(off[-1], R)):
        x[rows], g[rows], res[rows] = float('nan'), float('nan'), float('nan')
    for act in (None, 'silu'):
        leaves = [t.to(d).requires_grad_() for t in (x, w, b)]
        poison((R, N), (R, K), dt=dt)
        y = mhk.expert_dense(*leaves[:2], torch.tensor(off, dtype=torch.int32, device=d), leaves[2], act, res.to(d))
        poison((R, N), (R, K), dt=dt)
        grads = torch.autograd.grad(y, leaves, g.to(d))
        for rows in (slice(0, lead), slice(off[-1], R)):
            assert (y[rows] == 0).all() and (grads[0][rows] == 0).all(), (act, rows)
        for e, (i, j) in enumerate(zip(off, off[1:])):
            want = dense_case(x[i:j], w[e], b[e], act, res[i:j], g[i:j], dt)
            for name, t in zip(('y', 'dx', 'dw', 'db'), (y[i:j], grads[0][i:j], grads[1][e], grads[2][e])):
                near(f'{name} of {e}', t, *want[name])


@TYPES
def test_rows_before_the_first_group(dt, monkeypatch):
    for tile in [*matmul.tiles(dt), *matmul.FEW]:
        print(f'[case] leading rows, tile {tile} {dt}', flush=True)
        main = 'slow64' if tile in matmul.FEW else tile
        monkeypatch.setattr(matmul, '_choose_tile', lambda *a: main)
        monkeypatch.setattr(matmul, '_outer_plan', lambda R, M, N, groups, grouped, *a: (main, 128, -(-R // 128) + 3 * grouped))
        monkeypatch.setattr(matmul, '_few_tile', lambda *a: tile if tile in matmul.FEW else None)
        matmul._fwd_plan.cache_clear()
        try:
            _behind_leading_rows(dt)
        finally:
            monkeypatch.undo()
            matmul._fwd_plan.cache_clear()


def test_rows_before_the_first_group_by_halves(by_halves):  # noqa: F811
    print('[case] leading rows by halves', flush=True)
    _behind_leading_rows(F32)


@TYPES
def test_a_slice_of_the_experts(dt):
    """The offsets and weights of some of the experts give these experts' rows, by the sizes' own choice of kernels."""
    d = dev()
    print(f'[case] a slice of the experts {dt}', flush=True)
    rng = np.random.default_rng(5)
    T, E, K, N = 60, 6, 40, 24
    order = mhk.expert_order(torch.tensor(rng.integers(0, E, (T, 2)), device=d), E)
    x, w = rand(rng, T, K, dt=dt).to(d), rand(rng, E, N, K, dt=dt).to(d)
    rows = mhk.dispatch(x, order)
    whole = mhk.expert_dense(rows, w, order.offsets, activation='relu')
    poison((2 * T, N), dt=dt)
    part = mhk.expert_dense(rows, w[2:5], order.offsets[2:6], activation='relu')
    a, z = order.offsets[2].item(), order.offsets[5].item()
    assert torch.equal(part[a:z], whole[a:z]) and (part[:a] == 0).all() and (part[z:] == 0).all()


@pytest.mark.parametrize('dt', [F32, BF16], ids=['f32', 'bf16'])
def test_every_product_takes_the_same_rows_for_a_group(dt, monkeypatch):
    """Offsets that decrease: a row belongs to the group that the forward gives it in every gradient too, whether sums over rows
    are cut into pieces or not."""
    d = dev()
    rng = np.random.default_rng(12)
    R, K, N = 60, 24, 16
    x, w, b, g = rand(rng, R, K, dt=dt), rand(rng, 3, N, K, dt=dt), rand(rng, 3, N, dt=dt), rand(rng, R, N, dt=dt)
    off = torch.tensor([-4, 10, 5, 50], dtype=torch.int32, device=d)       # rows 0 to 9, none, 10 to 49
    for L, slots in ((0, 3), (64, 4)):
        print(f'[case] decreasing offsets {dt} L={L}', flush=True)
        monkeypatch.setattr(matmul, '_outer_plan', lambda *a: ('slow64', L, slots))
        matmul._bwd_plan.cache_clear()
        try:
            leaves = [t.to(d).requires_grad_() for t in (x, w, b)]
            y = mhk.expert_dense(*leaves[:2], off, leaves[2], 'silu')
            grads = torch.autograd.grad(y, leaves, g.to(d))
        finally:
            monkeypatch.undo()
            matmul._bwd_plan.cache_clear()
        assert (y[50:] == 0).all() and (grads[0][50:] == 0).all() and (grads[1][1] == 0).all() and (grads[2][1] == 0).all()
        for e, i in ((0, slice(0, 10)), (2, slice(10, 50))):
            want = dense_case(x[i], w[e], b[e], 'silu', None, g[i], dt)
            for name, t in zip(('y', 'dx', 'dw', 'db'), (y[i], grads[0][i], grads[1][e], grads[2][e])):
                near(f'{name} of {e}', t, *want[name])


# ------------------------------------------------------------------------------------------ operands that a tile cannot take
def test_the_library_holds_operands_to_whole_steps():
    """Modules of tiles straight to LDS refuse, before any launch, addresses and distances of rows that such loads cannot
    take.  (Operands here are of one row, so that no distance would lead out of them.)"""
    d = dev()
    print('[case] whole steps', flush=True)
    lib = _native.load()
    t, out = torch.ones(1 << 12, dtype=BF16, device=d), torch.zeros(64, 64, dtype=BF16, device=d)
    p, c, far = t.data_ptr(), out.data_ptr(), matmul.LD_MAX
    for tile in matmul.FAST:
        rows = matmul.module(d, BF16, 'fwd', tile).handle
        outer = matmul.module(d, BF16, 'dw', tile).handle

        def fwd(a, lda, b, ldb):
            return lib.mh_mm_rows(rows, a, lda, b, ldb, c, None, None, 0, None, None, 1, 1, 64, 1, _native.stream_of(t))

        def dw(a, lda, b, ldb):
            return lib.mh_mm_outer(outer, a, lda, b, ldb, c, None, None, 1, 64, 64, 1, 0, 1, _native.stream_of(t))

        for call in (fwd, dw):
            for args in ((p + 2, 64, p, 64), (p, 64, p + 8, 64), (p, 68, p, 64), (p, 64, p, 65), (p, far, p, 64), (p, 64, p, far)):
                assert call(*args) != 0 and 'whole steps' in lib.mh_last_error().decode(), (tile, call, args)
        assert fwd(p, 64, p, 64) == 0 and out[0, 0].item() == 64
        assert dw(p, far - 8, p, 64) == 0 and (out == 1).all()
        out.zero_()


# ------------------------------------------------------------------------------------------ forward-mode derivatives
def test_forward_mode_derivatives_are_refused():
    d = dev()
    print('[case] forward mode', flush=True)
    x, w = torch.randn(6, 8, device=d), torch.randn(8, 8, device=d)
    o = mhk.expert_order(torch.zeros(6, 1, dtype=torch.int64, device=d), 1)
    off = torch.tensor([0, 6], dtype=torch.int32, device=d)
    with torch.autograd.forward_ad.dual_level():
        t = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        v = torch.autograd.forward_ad.make_dual(w, torch.ones_like(w))
        for call in (lambda: mhk.dense(t, w), lambda: mhk.dense(x, v, activation='silu'), lambda: mhk.dense(x, w, residual=t),
                     lambda: mhk.dense(x, w, bias=v[0]), lambda: mhk.expert_dense(t, w[None], off),
                     lambda: mhk.dispatch(t, o), lambda: mhk.combine(t, None, o), lambda: mhk.combine(x, None, o, residual=t),
                     lambda: mhk.combine(x, t[:, :1], o), lambda: mhk.block_norm(t), lambda: mhk.block_norm(x, t),
                     lambda: mhk.block_norm(x, x, gate=t), lambda: mhk.block_norm(x, pre_weight=v[0])):
            for want in (False, True):
                w.requires_grad_(want)
                with pytest.raises((RuntimeError, NotImplementedError), match='forward-mode'):
                    call()
        w.requires_grad_(False)
        assert mhk.dense(x, w).shape == (6, 8)               # tensors without a tangent are taken as ever


# ------------------------------------------------------------------------------------------ slopes in an activation's tail
@pytest.mark.parametrize('dt', [BF16, F16], ids=['bf16', 'f16'])
@pytest.mark.parametrize('act', ['silu', 'gelu'])
@pytest.mark.parametrize('T', [50, 700])
def test_gradients_of_units_in_the_tail(T, act, dt):
    """Pre-activations between -4 and -12, where act' is down to 1e-30: gradients are right relative to their own size.

    Relative errors of a slope: 2^-9 by its coding, 3e-4 by its evaluation (of which 2.2e-4 the approximation of erf, the most
    that it is off in the tail), and that of its argument, whose error is (K + 16) 2^-24 of the magnitudes, times |act''/act'| <=
    |a| + 1.  Slopes below 2^-54 may come out as zero (float16 rounds their products to zero anyway)."""
    d = dev()
    print(f'[case] tail T={T} {act} {dt}', flush=True)
    rng = np.random.default_rng(9)
    K, N = 16, 72
    x, w, b = rand(rng, T, K, dt=dt), rand(rng, N, K, dt=dt, scale=0.02), torch.linspace(-4, -12, N).to(dt)
    g = (rand(rng, T, N) * 0.2 + 1).to(dt)
    leaves = [t.to(d).requires_grad_() for t in (x, w, b)]
    y = mhk.dense(*leaves[:2], leaves[2], act)
    dx, dw, db = (t.double().cpu() for t in torch.autograd.grad(y, leaves, g.to(d)))
    x, w, b, g = (t.double() for t in (x, w, b, g))
    a = x @ w.t() + b
    if act == 'silu':
        q = 1 / (1 + torch.exp(-a))
        slope = q * (1 + a * (1 - q))
    else:
        slope = 0.5 * torch.erfc(-a * 0.5 ** 0.5) + a * torch.exp(-0.5 * a * a) * (2 * np.pi) ** -0.5
    rel = 2.0 ** -9 + 3e-4 + (K + 16) * E32 * (x.abs() @ w.abs().t() + b.abs()) * (a.abs() + 1)
    p = g * slope
    err = p.abs() * (rel + E32) + g * 2.0 ** -54
    near('db', db, p.sum(0), err.sum(0) + ((T + 16) * E32 + U[dt]) * p.abs().sum(0) + TINY[dt])
    err = err + U[dt] * p.abs() + TINY[dt]                   # p rounded for the products
    for name, got, val, e, n in (('dx', dx, p @ w, (err @ w.abs(), p.abs() @ w.abs()), N),
                                 ('dw', dw, p.t() @ x, (err.t() @ x.abs(), p.abs().t() @ x.abs()), T)):
        near(name, got, val, e[0] + (n + 16) * E32 * e[1] + U[dt] * (val.abs() + e[0]) + TINY[dt])


# ------------------------------------------------------------------------------------------ unlike magnitudes
def _products(x, w, g, scale=None):
    """y, dx and dw of float32 tensors within the bound of a float32 sum: (n + 16) 2^-24 of the magnitudes added."""
    lx, lw = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = mhk.dense(lx, lw)
    dx, dw = torch.autograd.grad(y, (lx, lw), g.cuda())
    x, w, g = x.double(), w.double(), g.double()
    for name, got, a, b in (('y', y, x, w.t()), ('dx', dx, g, w), ('dw', dw, g.t(), x)):
        near(name, got, a @ b, (a.shape[1] + 16) * E32 * (a.abs() @ b.abs()))


@pytest.mark.parametrize('power', [4, 5, 9])
@pytest.mark.parametrize('K', [64, 1024])
def test_contractions_of_unlike_magnitudes_by_halves(K, power, by_halves):  # noqa: F811
    """Operands whose magnitudes along the contraction are each other's inverse, in units that differ by up to 10^18: every
    product counts alike, however small its factor is in its row."""
    dev()
    print(f'[case] unlike magnitudes K={K} power={power}', flush=True)
    rng = np.random.default_rng(K + power)
    T, N = 200, 160
    s = torch.logspace(-power, power, K)[torch.randperm(K, generator=torch.Generator().manual_seed(1))]
    _products(rand(rng, T, K) * s, rand(rng, N, K) / s, rand(rng, T, N))
    s = torch.logspace(-power, power, N)
    _products(rand(rng, T, K), rand(rng, N, K) / s[:, None], rand(rng, T, N) * s)
    s = torch.logspace(-power, power, T)
    _products(rand(rng, T, K) / s[:, None], rand(rng, N, K), rand(rng, T, N) * s[:, None])


@pytest.mark.parametrize('size', [1e8, 1e10, 1e20])
def test_one_large_value_by_halves(size, by_halves):  # noqa: F811
    """A value far above its row's others that meets a weight of zero leaves the others' sum its accuracy."""
    d = dev()
    print(f'[case] one value of {size}', flush=True)
    rng = np.random.default_rng(3)
    T, K, N = 150, 300, 140
    x, w, g = rand(rng, T, K), rand(rng, N, K), rand(rng, T, N)
    x[7, 5], x[90, 250], w[33, 7], g[50, 60] = size, -size, size, size
    w[::2, 5], w[1::2, 250], x[::2, 7], w[60, ::3], x[50, ::2] = 0, 0, 0, 0, 0
    _products(x, w, g)
    off = torch.tensor([0, 100, 150], dtype=torch.int32, device=d)
    lx, lw = x.to(d).requires_grad_(), torch.stack([w, w.flip(0)]).to(d).requires_grad_()
    y = mhk.expert_dense(lx, lw, off)
    dx, dw = torch.autograd.grad(y, (lx, lw), g.to(d))
    for e, (i, j) in enumerate(((0, 100), (100, 150))):
        a, b, c = x[i:j].double(), lw[e].detach().cpu().double(), g[i:j].double()
        for name, got, l, r in (('y', y[i:j], a, b.t()), ('dx', dx[i:j], c, b), ('dw', dw[e], c.t(), a)):
            near(f'{name} of {e}', got, l @ r, (l.shape[1] + 16) * E32 * (l.abs() @ r.abs()))


def test_rows_of_zeros_are_not_computed_again_by_halves(by_halves):  # noqa: F811
    """Zeros from rows or columns of zeros are right whatever the other operand holds; sums that cancel beside it are not."""
    d = dev()
    print('[case] rows of zeros', flush=True)
    rng = np.random.default_rng(6)
    T, K, N = 300, 64, 130
    x, w = rand(rng, T, K), rand(rng, N, K)
    x[::2], w[::3] = 0, 0
    w[1, 3] = 1e-25                                          # a wide row
    for again, x0 in ((False, x), (True, torch.cat([x[:-1], torch.tensor([[1e15] + [0.0] * (K - 2) + [1e-9]])]))):
        w[:, 0] = 0 if again else w[:, 0]
        words = torch.zeros(T + 1, dtype=torch.int32, device=d)
        y = torch.empty(T, N, device=d)
        h, c = (torch.empty(n, 2 * K, dtype=torch.int16, device=d) for n in (T, N))
        cw = torch.zeros(N + 1, dtype=torch.int32, device=d)
        xd, wd, s = x0.to(d), w.to(d), _native.stream_of(y)
        lib, split, mod = _native.load(), halves.module(d, 'split').handle, halves.module(d, 'fwd').handle
        P = lambda t: t.data_ptr()  # noqa: E731
        _native.check(lib.mh_hv_rows(split, P(xd), K, P(h), P(words), T, K, s))
        _native.check(lib.mh_hv_rows(split, P(wd), K, P(c), P(cw), N, K, s))
        _native.check(lib.mh_hv_mm(mod, P(h), P(c), P(y), None, None, 0, None, None, P(words), P(cw), None, T, N, K, 1, s))
        assert bool(words[T]) == again and (words[:T] >> 30 & 1).nonzero().flatten().tolist() == ([T - 1] if again else [])
    near('y', mhk.dense(xd, wd), x0.double() @ w.double().t(), (K + 16) * E32 * (x0.double().abs() @ w.double().abs().t()))


def test_infinities_that_meet_small_values_by_halves(by_halves):  # noqa: F811
    """An infinity times any other value than zero is infinite, however small that is in its row."""
    d = dev()
    print('[case] infinities and small values', flush=True)
    rng = np.random.default_rng(4)
    T, K, N = 150, 96, 140
    x, w = rand(rng, T, K), rand(rng, N, K)
    w[:, 5] = torch.where(torch.arange(N) % 2 == 0, 1e-30, -1e-25)
    w[3, 5] = 0
    x[2, 5], x[100, 5] = float('inf'), float('-inf')
    got, want = mhk.dense(x.to(d), w.to(d)).cpu(), (x.double() @ w.double().t())
    assert torch.isnan(want[2, 3]) and torch.isinf(want[2, :3]).all()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[[2, 100]].double().nan_to_num(7), want[[2, 100]].nan_to_num(7))


def test_products_by_halves_in_a_captured_graph(by_halves):  # noqa: F811
    """A captured forward and backward, replayed over inputs with and without values that the halves do not hold: every replay
    gives what the same calls give, and nothing of the replay before."""
    d = dev()
    print('[case] halves in a graph', flush=True)
    torch.manual_seed(3)
    T, K, N = 200, 96, 160
    x, w = torch.randn(T, K, device=d, requires_grad=True), torch.randn(N, K, device=d, requires_grad=True)
    g = torch.randn(T, N, device=d)

    def call():
        y = mhk.dense(x, w, activation='silu')
        return [y, *torch.autograd.grad(y, (x, w), g)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(6):
        with torch.no_grad():
            x.normal_()
            w.normal_()
            g.normal_()
            if i in (1, 2, 4):                               # not held: one value, one row, an infinity
                x[5, 7], w[:, 7] = (1e12, 0) if i != 4 else (float('inf'), 1e-20)
            if i == 2:
                g[:, 9] *= 1e-15
                g[3] *= 1e9
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, call()):
            assert torch.equal(a.nan_to_num(3), b.nan_to_num(3)), i
        if i != 4:
            want = dense_case(x.detach().cpu(), w.detach().cpu(), None, 'silu', None, g.cpu(), F32)
            for name, a in zip(('y', 'dx', 'dw'), out):
                near(f'{name} of replay {i}', a, *want[name])


# ------------------------------------------------------------------------------------------ many groups, many columns
def test_more_groups_than_a_grid_dimension_holds():
    d = dev()
    rng = np.random.default_rng(8)
    E, K, N = 70_001, 5, 3
    sizes = rng.integers(0, 3, E)
    off = torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=torch.int32)
    R = int(off[-1])
    e = torch.repeat_interleave(torch.arange(E), torch.tensor(sizes))
    for dt in (F32, BF16):
        for act in (None, 'relu'):
            print(f'[case] {E} groups {dt} {act}', flush=True)
            x, w, b, g = rand(rng, R, K, dt=dt), rand(rng, E, N, K, dt=dt), rand(rng, E, N, dt=dt), rand(rng, R, N, dt=dt)
            leaves = [t.to(d).requires_grad_() for t in (x, w, b)]
            y = mhk.expert_dense(*leaves[:2], off.to(d), leaves[2], act)
            dx, dw, db = torch.autograd.grad(y, leaves, g.to(d))
            a = (w.double()[e] @ x.double()[:, :, None])[:, :, 0] + b.double()[e]
            p = g.double() * ((a > 0) if act else 1)
            zero = torch.zeros(E, N, dtype=torch.float64)
            # five products of order one, rounded once (p is exact: a gradient or zero)
            near('y', y, ACTS[act](a), 40 * E32 * (a.abs() + 10) + U[dt] * (a.abs() + 1))
            near('dx', dx, (p[:, None] @ w.double()[e])[:, 0], 40 * E32 * 20 + U[dt] * (p[:, None] @ w.double()[e])[:, 0].abs())
            want = zero.index_add(0, e, p)
            near('db', db, want, 40 * E32 * 20 + U[dt] * want.abs())
            want = torch.zeros(E, N, K, dtype=torch.float64).index_add(0, e, p[:, :, None] * x.double()[:, None])
            near('dw', dw, want, 40 * E32 * 20 + U[dt] * want.abs())


def test_more_columns_than_a_grid_dimension_holds_workgroups():
    """Rows so wide that their pieces of 256 columns are more than 65,535."""
    d = dev()
    print('[case] wide rows', flush=True)
    N = 256 * 65535 + 300
    x = torch.tensor([[0.5, -2.0], [1.0, 3.0]], dtype=BF16, device=d, requires_grad=True)
    k = torch.arange(N, device=d)
    w = torch.stack([(k % 3).to(BF16), torch.ones_like(k, dtype=BF16)], 1).requires_grad_()
    b = (-(k % 2)).to(BF16).requires_grad_()
    y = mhk.dense(x, w, b, 'relu')
    a = x.detach().float() @ w.detach().float().t() + b.detach().float()              # small whole numbers and halves: exact
    assert torch.equal(y.float(), a.clamp_min(0))
    p = (a > 0).float()
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert torch.equal(db.float(), p.sum(0)) and torch.equal(dw.float(), p.t() @ x.detach().float())
    want = p.double() @ w.detach().double()
    near('dx', dx, want.cpu(), 2.0 ** -7 * want.abs().cpu())   # sums of up to 5 10^7 in some order, rounded to bfloat16


# ------------------------------------------------------------------------------------------ orders made by hand
def test_orders_that_expert_order_did_not_make_are_refused():
    """Places and offsets of another type, shape or layout are refused where the kernels would read past them."""
    d = dev()
    print('[case] orders by hand', flush=True)
    x = torch.zeros(6, 8, device=d)
    o = mhk.expert_order(torch.zeros(6, 2, dtype=torch.int64, device=d), 3)
    y = mhk.dispatch(x, o)
    for place, offsets in ((o.place[:1].expand(6, 2), o.offsets), (o.place.t().contiguous().t(), o.offsets),
                           (o.place.reshape(-1), o.offsets), (o.place.short(), o.offsets), (o.place, o.offsets.short()),
                           (o.place, o.offsets[:1].expand(4)), (o.place, o.offsets[None]), (o.place, o.offsets[:1]),
                           (o.place[:, :0].contiguous(), o.offsets)):
        bad = mhk.ExpertOrder(offsets, o.rows, place, 3)
        for call in (lambda: mhk.dispatch(x, bad), lambda: mhk.combine(y, None, bad)):
            with pytest.raises(ValueError, match='order'):
                call()
    again = mhk.ExpertOrder(o.offsets.clone(), o.rows, o.place.clone(), 3)
    assert torch.equal(mhk.dispatch(x, again), y) and mhk.combine(y, None, again).shape == (6, 8)


# ------------------------------------------------------------------------------------------ inputs given other data
def test_inputs_given_other_data_before_the_backward():
    """An input whose data was replaced between forward and backward, as moving a module to another device or type does, is
    refused; data of the same shape in another layout is read as it lies."""
    d = dev()
    print('[case] other data', flush=True)
    rng = np.random.default_rng(2)
    off = torch.tensor([0, 4, 6], dtype=torch.int32, device=d)
    o = mhk.expert_order(torch.tensor(rng.integers(0, 3, (6, 2)), device=d), 3)

    def leaves():
        return [rand(rng, *s).to(d).requires_grad_() for s in ((6, 8), (8, 8), (2, 8, 8), (8,), (12, 8), (6, 2), (6, 8))]

    layers = [(lambda x, w, ws, b, y, c, h: mhk.dense(x, w, b, 'silu'), (0, 1)),
              (lambda x, w, ws, b, y, c, h: mhk.expert_dense(x, ws, off), (0, 2)),
              (lambda x, w, ws, b, y, c, h: mhk.combine(y, c, o), (4, 5)),
              (lambda x, w, ws, b, y, c, h: mhk.block_norm(x, h, gate=x[:, :1], scale=b)[0], (0, 3, 6))]
    for call, used in layers:
        for i in used:
            for other in (lambda t: t.cpu(), lambda t: t.half(), lambda t: t.double(), lambda t: t[..., :1].contiguous()):
                ins = leaves()
                out = call(*ins)
                ins[i].data = other(ins[i].detach())
                with pytest.raises(RuntimeError, match='changed its shape|Expected|expected|same'):
                    out.sum().backward()
            ins = leaves()
            out = call(*ins)
            want = torch.autograd.grad(out.sum(), [ins[k] for k in used], retain_graph=True)
            ins[i].data = torch.stack([ins[i].detach()] * 2, -1)[..., 0]      # the same values, two apart
            got = torch.autograd.grad(out.sum(), [ins[k] for k in used])
            assert all(torch.equal(a, b) for a, b in zip(got, want)), i
