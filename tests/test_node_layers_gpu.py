"""
The trainable node layers (dense, expert_dense, expert_order, dispatch, combine, block_norm) against plain float64.

Tolerances are per element and follow from the arithmetic: a float32 sum of K products is off by at most
(K + 16) 2^-24 of the sum of their magnitudes (the 16 cover the parts of a split operand and the epilogue), an activation by
8 ulp, a rounding to the type by half a step: 2^-24, 2^-8 (bfloat16, 8 bits) or 2^-11 (float16, 11 bits, plus half its smallest step 2^-25) of the value,
and the kept slope of the 16-bit types by 2^-16.
"""
import numpy as np
import pytest
import torch

import mace_hip_kernels as mhk
from mace_hip_kernels import _native, halves, matmul, norms

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 0.0, BF16: 0.0, F16: 2.0 ** -25}
E32 = 2.0 ** -24
ACTS = {None: lambda a: a, 'relu': torch.relu, 'silu': torch.nn.functional.silu, 'gelu': torch.nn.functional.gelu}


def dev():
    assert torch.cuda.is_available(), 'GPU test needs a GPU'
    return torch.device('cuda:0')


def rand(rng, *shape, dt=F32, scale=1.0, mean=0.0):
    return torch.tensor(rng.standard_normal(shape) * scale + mean, dtype=torch.float64).to(dt)


def near(name, got, want, tol):
    got, want, tol = got.detach().double().cpu(), want.detach().double(), torch.as_tensor(tol, dtype=torch.float64)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f'{name}: NaN in other places'
    bad = ~((got - want).abs() <= tol) & ~torch.isnan(want) & (got != want)
    if bad.any():
        i = int(torch.argmax(((got - want).abs() / tol.expand_as(want).clamp_min(1e-300)).nan_to_num().reshape(-1)))
        raise AssertionError(f'{name}: {int(bad.sum())} of {bad.numel()} values off, worst at {i}: '
                             f'{got.reshape(-1)[i]:.9g} for {want.reshape(-1)[i]:.9g}, '
                             f'bound {tol.expand_as(want).reshape(-1)[i]:.3g}')


def dense_case(x, w, b, act, res, g, dt):
    """y, its gradients, and the bounds of all of them, in float64 on the CPU for inputs of type dt."""
    x, w = x.double(), w.double()
    T, K = x.shape
    N = w.shape[0]
    b64 = torch.zeros(N, dtype=torch.float64) if b is None else b.double()
    leaf = (x @ w.t() + b64).requires_grad_()
    y = ACTS[act](leaf)
    slope, = torch.autograd.grad(y.sum(), leaf)
    a, y = leaf.detach(), y.detach()
    mag = x.abs() @ w.abs().t() + b64.abs()
    err_a = (K + 16) * E32 * mag
    err = 1.2 * err_a + 8 * E32 * (a.abs() + 1) * (act not in (None, 'relu'))
    if res is not None:
        y = y + res.double()
    want = dict(y=(y, err + (U[dt] + E32) * (y.abs() + err) + TINY[dt] + E32 * (0 if res is None else res.double().abs())))
    if g is None:
        return want
    g = g.double()
    p = g * slope
    # slope: its argument's error (|act''| < 1.2; a relu may switch where a is within its error of 0), evaluation, storage
    err_s = (1.2 * err_a + 16 * E32 + (0 if dt == F32 else 2.0 ** -16)) * (act not in (None, 'relu'))
    if act == 'relu':
        err_s = (a.abs() <= err_a).double()
    err_p = g.abs() * err_s + E32 * p.abs()
    want['db'] = (p.sum(0), err_p.sum(0) + (T + 16) * E32 * p.abs().sum(0) + U[dt] * p.sum(0).abs() + TINY[dt])
    err_q = err_p + (U[dt] * p.abs() + TINY[dt] if act is not None else 0)
    for name, val, mags, n in (('dx', p @ w, (p.abs(), w.abs(), err_q), N), ('dw', p.t() @ x, (p.abs().t(), x.abs(), err_q.t()), T)):
        e = (n + 16) * E32 * (mags[0] @ mags[1]) + mags[2] @ mags[1]
        want[name] = (val, e + (U[dt] + E32) * (val.abs() + e) + TINY[dt])
    return want


DENSE = [(1, 1, 1), (1, 64, 128), (3, 7, 5), (16, 32, 64), (17, 33, 65), (64, 128, 256), (129, 515, 131), (300, 100, 40),
         (1, 1024, 513), (5, 1027, 70), (33, 2048, 24), (700, 9, 300)]


@pytest.mark.parametrize('dt', [F32, BF16, F16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('T,K,N', DENSE)
def test_dense_and_its_gradients(T, K, N, dt):
    d = dev()
    rng = np.random.default_rng(T * 7919 + K * 31 + N)
    for act in (None, 'relu', 'silu', 'gelu'):
        print(f'[case] dense T={T} K={K} N={N} {dt} {act}', flush=True)
        x, w, b = rand(rng, T, K, dt=dt), rand(rng, N, K, dt=dt, scale=K ** -0.5), rand(rng, N, dt=dt)
        res = rand(rng, T, N, dt=dt) if act in ('silu', None) else None
        g = rand(rng, T, N, dt=dt)
        want = dense_case(x, w, b, act, res, g, dt)
        leaves = [t.to(d).requires_grad_() for t in (x, w, b)]
        r = None if res is None else res.to(d).requires_grad_()
        y = mhk.dense(*leaves[:2], bias=leaves[2], activation=act, residual=r)
        grads = torch.autograd.grad(y, leaves + ([r] if r is not None else []), g.to(d))
        plain = mhk.dense(*(t.detach() for t in leaves[:2]), bias=leaves[2].detach(), activation=act,
                          residual=None if r is None else r.detach())
        near('y', y, *want['y'])
        near('y without gradients', plain, *want['y'])
        for name, t in zip(('dx', 'dw', 'db'), grads):
            near(name, t, *want[name])
        if r is not None:
            assert torch.equal(grads[3].cpu(), g)


@pytest.mark.parametrize('T,K,N,dt', [(2600, 256, 640, F32), (5000, 128, 96, BF16), (2500, 1024, 1536, BF16),
                                      (2048, 256, 2304, F16), (9000, 72, 200, F16), (20000, 64, 64, F32)])
def test_dense_over_many_tiles_and_split_sums(T, K, N, dt):
    d = dev()
    print(f'[case] dense T={T} K={K} N={N} {dt}', flush=True)
    rng = np.random.default_rng(5)
    x, w, b, g = rand(rng, T, K, dt=dt), rand(rng, N, K, dt=dt, scale=K ** -0.5), rand(rng, N, dt=dt), rand(rng, T, N, dt=dt)
    want = dense_case(x, w, b, 'silu', None, g, dt)
    leaves = [t.to(d).requires_grad_() for t in (x, w, b)]
    y = mhk.dense(*leaves[:2], bias=leaves[2], activation='silu')
    first = torch.autograd.grad(y, leaves, g.to(d), retain_graph=True)
    near('y', y, *want['y'])
    for name, t, u in zip(('dx', 'dw', 'db'), first, torch.autograd.grad(y, leaves, g.to(d))):
        near(name, t, *want[name])
        assert torch.equal(t, u), f'{name} differs between two passes'


@pytest.fixture
def by_halves(monkeypatch):
    """Float32 products by halves whatever their size."""
    monkeypatch.setattr(halves, 'pays', lambda *a: True)
    matmul._fwd_plan.cache_clear()
    matmul._bwd_plan.cache_clear()
    yield
    monkeypatch.undo()
    matmul._fwd_plan.cache_clear()
    matmul._bwd_plan.cache_clear()


@pytest.mark.parametrize('T,K,N', DENSE + [(260, 328, 520), (2600, 40, 136)])
def test_products_by_halves(T, K, N, by_halves):
    d = dev()
    rng = np.random.default_rng(T + K)
    cuts = [T // 3, T // 3, T - T // 5]
    off = torch.tensor([0] + cuts, dtype=torch.int32)
    for act in (None, 'gelu'):
        print(f'[case] halves T={T} K={K} N={N} {act}', flush=True)
        x, w, b, g = rand(rng, T, K), rand(rng, 3, N, K, scale=K ** -0.5), rand(rng, 3, N), rand(rng, T, N)
        res = rand(rng, T, N)
        x[cuts[2]:], g[cuts[2]:] = 1e30, float('nan')              # rows of no group
        one = dense_case(x[:cuts[2]], w[0], b[0], act, res[:cuts[2]], g[:cuts[2]], F32)
        leaves = [t.to(d).requires_grad_() for t in (x, w, b)]
        y = mhk.dense(leaves[0][:cuts[2]], leaves[1][0], leaves[2][0], act, res[:cuts[2]].to(d))
        near('y', y, *one['y'])
        grads = torch.autograd.grad(y, leaves, g[:cuts[2]].to(d))
        for name, t in zip(('dx', 'dw', 'db'), (grads[0][:cuts[2]], grads[1][0], grads[2][0])):
            near(name, t, *one[name])
        y = mhk.expert_dense(*leaves[:2], off.to(d), leaves[2], act, res.to(d))
        grads = torch.autograd.grad(y, leaves, g.to(d))
        assert (y[cuts[2]:] == 0).all() and (grads[0][cuts[2]:] == 0).all()
        for e, (i, j) in enumerate(zip([0] + cuts[:2], cuts)):
            want = dense_case(x[i:j], w[e], b[e], act, res[i:j], g[i:j], F32)
            for name, t in zip(('y', 'dx', 'dw', 'db'), (y[i:j], grads[0][i:j], grads[1][e], grads[2][e])):
                near(f'{name} of {e}', t, *want[name])


def _odd_values(path):
    """Infinities and NaN in x, the weight and the gradient reach what they reach in a float32 sum, and nothing else; rows
    and columns of very different magnitudes keep float32 accuracy each."""
    d = dev()
    print(f'[case] odd values, {path}', flush=True)
    rng = np.random.default_rng(21)
    T, K, N = 200, 96, 160
    x, w, g = rand(rng, T, K), rand(rng, N, K), rand(rng, T, N)
    x = x * torch.logspace(-18, 18, T)[:, None]
    w = w * torch.logspace(-9, 9, N)[:, None]
    want = dense_case(x, w, None, None, None, None, F32)
    near('y', mhk.dense(x.to(d), w.to(d)), *want['y'])
    x, w = rand(rng, T, K) * torch.logspace(-15, 12, K), rand(rng, N, K) * torch.logspace(-9, 9, K)
    g = rand(rng, T, N) * torch.logspace(-12, 9, N)
    want = dense_case(x, w, None, None, None, g, F32)
    lx, lw = x.to(d).requires_grad_(), w.to(d).requires_grad_()
    dx, dw = torch.autograd.grad(mhk.dense(lx, lw), (lx, lw), g.to(d))
    near('dw', dw, *want['dw'])
    near('dx', dx, *want['dx'])
    x, w, g = rand(rng, T, K), rand(rng, N, K), rand(rng, T, N)
    w[:, 5], w[3, 5], w[4, 5] = 1.0, 0.0, -2.0
    x[0, 5], x[150, 5], x[1, 7], w[9, 11] = float('inf'), float('-inf'), float('nan'), float('inf')
    g[7, 9], g[8, 10], g[9, 140] = float('nan'), float('inf'), float('-inf')
    for name, got, want in (('y', mhk.dense(x.to(d), w.to(d)), x.double() @ w.double().t()),):
        odd = ~torch.isfinite(want)
        assert odd[0].all() and torch.isinf(want[0, 0]) and torch.isnan(want[0, 3]) and not odd[2, 0]
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want)), name
        inf = odd & ~torch.isnan(want)
        assert torch.equal(got.cpu().double()[inf], want[inf]), name
        near(name, got.cpu()[~odd], want[~odd], (K + 16) * E32 * (x.nan_to_num(0, 0, 0).double().abs()
                                                                  @ w.nan_to_num(0, 0, 0).double().abs().t())[~odd])
    x, w = x.nan_to_num(0.5, 0.5, 0.5), w.nan_to_num(0.5, 0.5, 0.5)
    lx, lw = x.to(d).requires_grad_(), w.to(d).requires_grad_()
    dx, dw = torch.autograd.grad(mhk.dense(lx, lw), (lx, lw), g.to(d))
    for name, got, want, odd in (('dx', dx, g.double() @ w.double(), [7, 8, 9]), ('dw', dw, g.double().t() @ x.double(), [9, 10, 140])):
        got = got.cpu()
        rest = [i for i in range(len(want)) if i not in odd]
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.isfinite(got[rest]).all(), name
        inf = torch.isinf(want)
        assert inf.any() and torch.equal(got.double()[inf], want[inf]), name


def test_odd_values_direct():
    _odd_values('direct')


def test_odd_values_by_halves(by_halves):
    _odd_values('halves')


@pytest.mark.parametrize('T,K,N', [(300, 200, 264), (1, 8, 8), (513, 64, 72), (260, 328, 520), (301, 203, 131), (140, 1, 7)])
@pytest.mark.parametrize('dt', [F32, BF16, F16], ids=['f32', 'bf16', 'f16'])
def test_every_tile(T, K, N, dt, monkeypatch):
    """Each tile in all three products, one and three groups with a tail, whatever the sizes would have chosen."""
    d = dev()
    rng = np.random.default_rng(T)
    cuts = sorted(rng.integers(0, T + 1, 3).tolist())
    x, w, b, g = rand(rng, T, K, dt=dt), rand(rng, 3, N, K, dt=dt, scale=K ** -0.5), rand(rng, 3, N, dt=dt), rand(rng, T, N, dt=dt)
    off = torch.tensor([0] + cuts, dtype=torch.int32)
    one = dense_case(x, w[0], b[0], 'silu', None, g, dt)
    three = [dense_case(x[i:j], w[e], b[e], 'silu', None, g[i:j], dt) for e, (i, j) in enumerate(zip([0] + cuts[:2], cuts))]
    def choose(tile):
        main = 'slow64' if tile in matmul.FEW else tile
        fast = main in matmul.FAST                       # copies to whole steps of 16 bytes where a shape needs them
        monkeypatch.setattr(matmul, '_choose_tile', lambda *a: main)
        monkeypatch.setattr(matmul, '_outer_plan', lambda R, M, N, groups, grouped, *a: (main, 128, -(-R // 128) + 3 * grouped))
        monkeypatch.setattr(matmul, '_few_tile', lambda *a: tile if tile in matmul.FEW else None)
        monkeypatch.setattr(matmul, '_padding_pays', lambda *a: fast)
        matmul._fwd_plan.cache_clear()
        matmul._bwd_plan.cache_clear()

    for tile in [*matmul.tiles(dt), *matmul.FEW]:
        print(f'[case] tile {tile} T={T} K={K} N={N} {dt}', flush=True)
        choose(tile)
        leaves = [t.to(d).requires_grad_() for t in (x, w, b)]
        y = mhk.dense(leaves[0], leaves[1][0], leaves[2][0], 'silu')
        near('y', y, *one['y'])
        grads = torch.autograd.grad(y, leaves, g.to(d))
        for name, t in zip(('dx', 'dw', 'db'), (grads[0], grads[1][0], grads[2][0])):
            near(name, t, *one[name])
        y = mhk.expert_dense(*leaves[:2], off.to(d), leaves[2], 'silu')
        grads = torch.autograd.grad(y, leaves, g.to(d))
        assert (y[cuts[2]:] == 0).all() and (grads[0][cuts[2]:] == 0).all()
        for e, want in enumerate(three):
            i = slice(int(off[e]), int(off[e + 1]))
            for name, t in zip(('y', 'dx', 'dw', 'db'), (y[i], grads[0][i], grads[1][e], grads[2][e])):
                near(f'{name} of {e}', t, *want[name])
    monkeypatch.undo()
    matmul._fwd_plan.cache_clear()
    matmul._bwd_plan.cache_clear()


@pytest.mark.parametrize('dt', [F32, BF16], ids=['f32', 'bf16'])
def test_dense_takes_strides_leading_dimensions_and_no_rows(dt):
    d = dev()
    rng = np.random.default_rng(11)
    wide, w = rand(rng, 6, 10, 150, dt=dt).to(d), rand(rng, 40, 70, dt=dt).to(d)
    for name, x in (('a slice of wider rows', wide[..., 40:110]), ('transposed', rand(rng, 70, 12, dt=dt).to(d).t()),
                    ('one row repeated', rand(rng, 1, 70, dt=dt).to(d).expand(9, 70)),
                    ('every second column', rand(rng, 5, 140, dt=dt).to(d)[:, ::2])):
        print(f'[case] dense strides: {name} {dt}', flush=True)
        res = rand(rng, *x.shape[:-1], 80, dt=dt).to(d)[..., 20:60]
        x1 = x.detach().requires_grad_()
        y = mhk.dense(x1, w.t().contiguous().t(), residual=res, activation='relu')
        want = dense_case(x.reshape(-1, 70).cpu(), w.cpu(), None, 'relu', res.reshape(-1, 40).cpu(),
                          torch.ones(y.numel() // 40, 40, dtype=dt), dt)
        assert y.shape == (*x.shape[:-1], 40)
        near('y', y.reshape(-1, 40), *want['y'])
        gx, = torch.autograd.grad(y.sum(), x1)            # an expanded gradient
        near('dx', gx.reshape(-1, 70), *want['dx'])
    print(f'[case] dense without rows or columns {dt}', flush=True)
    for T, K, N in ((0, 8, 4), (3, 0, 4), (3, 8, 0)):
        x, w = (torch.ones(T, K, dtype=dt, device=d).requires_grad_(), torch.ones(N, K, dtype=dt, device=d).requires_grad_())
        b = torch.ones(N, dtype=dt, device=d).requires_grad_()
        y = mhk.dense(x, w, b)
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
        assert y.shape == (T, N) and gx.shape == x.shape and (gb == T).all() and (gw == T).all() and (gx == N).all()
        assert (y == K + 1).all()


@pytest.mark.parametrize('dt', [F32, BF16, F16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('T', [2, 40])
def test_dense_infinities_and_nan_act_as_in_a_plain_sum(dt, T):
    d = dev()
    print(f'[case] dense with infinities {dt} T={T}', flush=True)
    K, N = 96, 80
    rng = np.random.default_rng(2)
    x, w = rand(rng, T, K, dt=dt), rand(rng, N, K, dt=dt)
    w[:, 5] = 1.0                                    # exact in 8 bits: its lower parts are zero
    w[3, 5] = 0.0
    w[4, 5] = -2.0
    x[0, 5] = float('inf')
    x[1, 7] = float('nan')
    w[9, 11] = float('inf')
    y = mhk.dense(x.to(d), w.to(d)).cpu()
    want = x.double() @ w.double().t()
    assert torch.isinf(want[0, 0]) and torch.isnan(want[0, 3])
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    assert torch.equal(y.double()[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)])
    assert torch.isfinite(y[~odd]).all()
    a = torch.tensor([[float('nan'), 0.0, -1.0]], dtype=dt, device=d)
    eye = torch.eye(3, dtype=dt, device=d)
    a[0, 1:] = 0.0
    assert torch.isnan(mhk.dense(a, eye, activation='relu')[0, 0])


def test_dense_wide_range_of_float32():
    """Rows of very different magnitude keep float32 accuracy each."""
    d = dev()
    print('[case] dense range', flush=True)
    rng = np.random.default_rng(8)
    x, w = rand(rng, 40, 64), rand(rng, 24, 64)
    x = x * torch.logspace(-30, 30, 40)[:, None]
    want = dense_case(x, w, None, None, None, None, F32)
    near('y', mhk.dense(x.to(d), w.to(d)), *want['y'])


# ---------------------------------------------------------------------------------------------------- experts' products
GROUPS = [([5], 16, 24), ([0, 3, 0, 1], 33, 17), ([130, 1, 0, 64, 500], 64, 96), ([1] * 70, 40, 130), ([0, 0], 8, 8),
          ([300, 900, 2, 1500], 200, 136)]


@pytest.mark.parametrize('dt', [F32, BF16, F16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('sizes,K,N', GROUPS)
@pytest.mark.parametrize('tail', [0, 37])
def test_expert_dense_and_its_gradients(sizes, K, N, tail, dt):
    d = dev()
    print(f'[case] expert_dense sizes={sizes[:6]} K={K} N={N} tail={tail} {dt}', flush=True)
    rng = np.random.default_rng(len(sizes) * 100 + K + tail)
    E, n = len(sizes), sum(sizes)
    R = n + tail
    off = torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=torch.int32)
    x, w, b = rand(rng, R, K, dt=dt), rand(rng, E, N, K, dt=dt, scale=K ** -0.5), rand(rng, E, N, dt=dt)
    res, g = rand(rng, R, N, dt=dt), rand(rng, R, N, dt=dt)
    if tail:
        x[n:], g[n:], res[n:] = float('nan'), float('nan'), float('nan')     # rows of no group are not read
    act = 'gelu' if N == 96 else 'silu'
    leaves = [t.to(d).requires_grad_() for t in (x, w, b)]
    y = mhk.expert_dense(*leaves[:2], off.to(d), leaves[2], act, res.to(d))
    grads = torch.autograd.grad(y, leaves, g.to(d))
    assert (y[n:] == 0).all() and (grads[0][n:] == 0).all()
    for e in range(E):
        i = slice(int(off[e]), int(off[e + 1]))
        want = dense_case(x[i], w[e], b[e], act, res[i], g[i], dt)
        near(f'y of {e}', y[i], *want['y'])
        near(f'dx of {e}', grads[0][i], *want['dx'])
        near(f'dw of {e}', grads[1][e], *want['dw'])
        near(f'db of {e}', grads[2][e], *want['db'])


@pytest.mark.parametrize('dt', [F32, BF16], ids=['f32', 'bf16'])
def test_each_gradient_alone(dt):
    """Every subset of inputs with gradients gives the gradients that all together give."""
    d = dev()
    rng = np.random.default_rng(31)
    T, K, N, E = 90, 40, 48, 3
    x, w, b, r = rand(rng, T, K, dt=dt), rand(rng, E, N, K, dt=dt), rand(rng, E, N, dt=dt), rand(rng, T, N, dt=dt)
    g = rand(rng, T, N, dt=dt).to(d)
    off = torch.tensor([0, 20, 20, 85], dtype=torch.int32, device=d)
    for act in (None, 'silu'):
        print(f'[case] gradients alone {act} {dt}', flush=True)

        def run(mask):
            ts = [t.to(d).requires_grad_(m) for t, m in zip((x, w, b, r), mask)]
            outs = [mhk.expert_dense(ts[0], ts[1], off, ts[2], act, ts[3]),
                    mhk.dense(ts[0], ts[1][0], ts[2][0], act, ts[3])]
            ins = [t for t, m in zip(ts, mask) if m]
            return [torch.autograd.grad(y, ins, g) for y in outs]

        full = run((True,) * 4)
        for m in range(1, 15):
            mask = [bool(m >> i & 1) for i in range(4)]
            for got, want in zip(run(mask), full):
                for a, bb in zip(got, [t for t, q in zip(want, mask) if q]):
                    assert torch.equal(a, bb), (act, mask)
    o = mhk.expert_order(torch.randint(-1, 4, (T, 2), device=d), 4)
    y, wt, res = rand(rng, 2 * T, N, dt=dt), rand(rng, T, 2), rand(rng, T, N, dt=dt)

    def mix(mask):
        ts = [t.to(d).requires_grad_(m) for t, m in zip((y, wt, res), mask)]
        return torch.autograd.grad(mhk.combine(*ts[:2], o, ts[2]), [t for t, m in zip(ts, mask) if m], g)

    full = mix((True,) * 3)
    for m in range(1, 7):
        mask = [bool(m >> i & 1) for i in range(3)]
        for a, bb in zip(mix(mask), [t for t, q in zip(full, mask) if q]):
            assert torch.equal(a, bb), mask


@pytest.mark.parametrize('E', [64, 65, 200, 1000])
def test_expert_dense_over_many_groups(E):
    d = dev()
    print(f'[case] expert_dense of {E} groups', flush=True)
    rng = np.random.default_rng(E)
    sizes = rng.integers(0, 9, E) * (rng.random(E) < 0.7)
    sizes[E // 2] = 150
    off = torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=torch.int32)
    n, K, N = int(off[-1]), 24, 40
    x, w, g = rand(rng, n + 5, K, dt=BF16), rand(rng, E, N, K, dt=BF16), rand(rng, n + 5, N, dt=BF16)
    lx, lw = x.to(d).requires_grad_(), w.to(d).requires_grad_()
    y = mhk.expert_dense(lx, lw, off.to(d), activation='relu')
    dx, dw = torch.autograd.grad(y, (lx, lw), g.to(d))
    for e in (0, 1, E // 2, E - 2, E - 1):
        i = slice(int(off[e]), int(off[e + 1]))
        want = dense_case(x[i], w[e], None, 'relu', None, g[i], BF16)
        for name, t in (('y', y[i]), ('dx', dx[i]), ('dw', dw[e])):
            near(f'{name} of {e}', t, *want[name])
    assert (y[n:] == 0).all() and (dx[n:] == 0).all()


def test_tensors_past_32_bit_offsets():
    """Results and operands of more than 2^31 values: the rows behind that are as right as the first."""
    d = dev()
    print('[case] more than 2^31 values', flush=True)
    T, K, N = 1_050_000, 16, 2056
    assert T * N > 2 ** 31
    g = torch.Generator(device=d).manual_seed(1)
    x = torch.randn(T, K, generator=g, device=d).bfloat16().requires_grad_()
    w, b = torch.randn(N, K, generator=g, device=d).bfloat16(), torch.randn(N, generator=g, device=d).bfloat16()
    y = mhk.dense(x, w, b, 'silu')
    gy = torch.ones(1, 1, device=d, dtype=BF16).expand(T, N)
    dx, = torch.autograd.grad(y, x, gy)
    for i in (slice(0, 40), slice(T - 40, T)):
        want = dense_case(x.detach()[i].cpu(), w.cpu(), b.cpu(), 'silu', None, torch.ones(40, N, dtype=BF16), BF16)
        near('y', y[i], *want['y'])
        near('dx', dx[i], *want['dx'])
    h, n = mhk.block_norm(y, y, scale=b)
    want = norm_case(y[-40:].cpu(), y[-40:].cpu(), None, b.cpu(), None, None, None, None, 'rms', 1e-6)
    near('h', h[-40:], want['h'], 1e-5 * 64 + U[BF16] * want['h'].abs())
    del h, n
    e = torch.arange(T, device=d)[:, None] % 7
    o = mhk.expert_order(e, 7)
    xs = mhk.dispatch(y.detach(), o)
    assert torch.equal(xs[o.place[-3:, 0].long()], y[-3:])
    assert torch.equal(mhk.combine(xs, None, o)[-3:], y[-3:])


def test_expert_dense_with_offsets_out_of_range_stays_inside():
    """Contents of the offsets never lead out of the tensors: the call ends, and rows inside its groups are theirs."""
    d = dev()
    print('[case] expert_dense offsets out of range', flush=True)
    rng = np.random.default_rng(3)
    x, w = rand(rng, 50, 16).to(d).requires_grad_(), rand(rng, 3, 8, 16).to(d).requires_grad_()
    off = torch.tensor([-4, 10, 5, 900], dtype=torch.int32, device=d)
    y = mhk.expert_dense(x, w, off)
    torch.autograd.grad(y, (x, w), torch.ones_like(y))
    want = x[:10].double() @ w[0].double().t()
    assert (y[:5].double() - want[:5]).abs().max() < 1e-5


# ---------------------------------------------------------------------------------------------------- routing
def order_of(experts, E):
    flat = experts.reshape(-1).tolist()
    lists = [[i for i, e in enumerate(flat) if e == x] for x in range(E)]
    rows = [i for li in lists for i in li]
    place = [-1] * len(flat)
    for p, i in enumerate(rows):
        place[i] = p
    return np.cumsum([0] + [len(li) for li in lists]), rows + [-1] * (len(flat) - len(rows)), place


@pytest.mark.parametrize('T,k,E', [(0, 2, 4), (1, 1, 1), (1, 4, 7), (63, 1, 4), (160, 2, 64), (1025, 3, 5), (2100, 2, 1024),
                                   (6000, 1, 89), (5000, 4, 128), (9000, 2, 1023)])
@pytest.mark.parametrize('wide', [False, True])
def test_expert_order_is_the_stable_sort(T, k, E, wide):
    d = dev()
    print(f'[case] expert_order T={T} k={k} E={E} wide={wide}', flush=True)
    rng = np.random.default_rng(T + k + E)
    e = rng.integers(0, E, (T, k))
    drop = rng.random((T, k))
    e[drop < 0.1] = -1
    e[drop > 0.97] = E
    if wide:
        e[(drop > 0.5) & (drop < 0.52)] = 2 ** 32      # equal to 0 in its low half
    o = mhk.expert_order(torch.tensor(e, dtype=torch.int64 if wide else torch.int32, device=d), E)
    off, rows, place = order_of(e, E)
    assert o.offsets.tolist() == off.tolist()
    assert o.rows.tolist() == rows and o.place.reshape(-1).tolist() == place
    assert o.place.shape == (T, k)


@pytest.mark.parametrize('dt', [F32, BF16, F16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('T,k,E,C', [(1, 1, 1, 1), (1, 2, 4, 33), (160, 1, 4, 128), (301, 3, 9, 515), (77, 4, 128, 1031),
                                     (2500, 2, 8, 24), (40, 2, 3, 4100)])
def test_dispatch_and_combine_and_their_gradients(T, k, E, C, dt):
    d = dev()
    print(f'[case] dispatch, combine T={T} k={k} E={E} C={C} {dt}', flush=True)
    rng = np.random.default_rng(T + C)
    e = rng.integers(0, E, (T, k))
    e[rng.random((T, k)) < 0.15] = -1
    if T > 3:
        e[2] = -1                                        # a node that every expert dropped
    off, rows, place = order_of(e, E)
    place, n = torch.tensor(place).view(T, k), int(off[-1])
    kept = (place >= 0).double()
    at = place.clamp_min(0)
    x, y, w, res = rand(rng, T, C, dt=dt), rand(rng, T * k, C, dt=dt), rand(rng, T, k), rand(rng, T, C, dt=dt)
    y[n:] = float('nan')                                 # rows of no assignment, and dropped weights, are not read
    w[place < 0] = float('nan')
    gx, go = rand(rng, T * k, C, dt=dt), rand(rng, T, C, dt=dt)
    gx[n:] = float('nan')
    o = mhk.expert_order(torch.tensor(e, device=d), E)
    lx, ly, lw, lr = (t.to(d).requires_grad_() for t in (x, y, w, res))
    xs = mhk.dispatch(lx, o)
    src = torch.tensor(rows[:n], dtype=torch.long) // k
    assert torch.equal(xs[:n].cpu(), x[src]) and (xs[n:] == 0).all()
    out = mhk.combine(ly, lw, o, residual=lr)
    y64, w64 = y.double().nan_to_num(), w.double().nan_to_num() * kept
    terms = y64[at] * w64[..., None]
    val = terms.sum(1) + res.double()
    mag = terms.abs().sum(1) + res.double().abs()
    near('out', out, val, (k + 2) * E32 * mag + U[dt] * (val.abs() + (k + 2) * E32 * mag) + TINY[dt])
    dx, dy, dw, dr = torch.autograd.grad((xs, out), (lx, ly, lw, lr), (gx.to(d), go.to(d)))
    t = gx.double().nan_to_num()[at] * kept[..., None]
    near('dx', dx, t.sum(1), (k + 2) * E32 * t.abs().sum(1) + U[dt] * t.abs().sum(1) + TINY[dt])
    want = torch.zeros(T * k, C, dtype=torch.float64)
    want[:n] = go.double()[src] * w64.reshape(-1)[torch.tensor(rows[:n], dtype=torch.long)][:, None]
    near('dy', dy, want, (U[dt] + 2 * E32) * want.abs() + TINY[dt])
    prod = y64[at] * go.double()[:, None] * kept[..., None]
    near('dw', dw, prod.sum(2), (C + 16) * E32 * prod.abs().sum(2))
    assert torch.equal(dr.cpu(), go)
    only = mhk.combine(ly.detach(), None, o)              # no weights, no residual
    t = y64[at] * kept[..., None]
    near('sum', only, t.sum(1), (k + 2) * E32 * t.abs().sum(1) + U[dt] * t.abs().sum(1) + TINY[dt])


def test_routing_takes_strided_rows_and_weights_of_the_type():
    d = dev()
    print('[case] routing strides', flush=True)
    rng = np.random.default_rng(4)
    T, k, C = 50, 2, 24
    o = mhk.expert_order(torch.tensor(rng.integers(0, 5, (T, k)), device=d), 5)
    wide = rand(rng, T, 3 * C, dt=BF16).to(d)
    xs = mhk.dispatch(wide[:, C:2 * C], o)
    assert torch.equal(xs, mhk.dispatch(wide[:, C:2 * C].contiguous(), o))
    w = rand(rng, k, T, dt=BF16).to(d).t().requires_grad_()
    out = mhk.combine(xs, w, o, residual=wide[:, :C])
    assert torch.equal(out, mhk.combine(xs, w.detach().float(), o, residual=wide[:, :C].contiguous()))
    gw, = torch.autograd.grad(out.sum(), w)               # an expanded gradient
    assert gw.dtype == BF16 and gw.shape == (T, k)


# ---------------------------------------------------------------------------------------------------- norms
def norm_case(x, y, gate, s, wp, wn, gh, gn, kind, eps):
    """h, n and all gradients in float64 from the formulas (no autograd), for 2-D inputs."""
    def norm(v):
        if kind == 'layer':
            v = v - v.mean(1, keepdim=True)
        r = ((v * v).mean(1, keepdim=True) + eps).rsqrt()
        return v * r, r

    def back(g, v, r):
        d = g - v * (g * v).mean(1, keepdim=True)
        return r * (d - g.mean(1, keepdim=True) if kind == 'layer' else d)

    one = torch.ones(1, dtype=torch.float64)
    s, wp, wn, gate = (one if t is None else t.double() for t in (s, wp, wn, gate))
    x = x.double()
    out = {}
    if y is not None:
        u, ru = norm(y.double())
        h = x + s * gate * u * wp
    else:
        h = x
    v, rv = norm(h)
    out.update(h=h, n=v * wn)
    if gn is not None:
        gh, gn = gh.double(), gn.double()
        dh = (gh if y is not None else 0) + back(gn * wn, v, rv)
        out.update(dx=dh, dwn=(gn * v).sum(0))
        if y is not None:
            out.update(dy=back(dh * gate * s * wp, u, ru), ds=(dh * gate * u * wp).sum(0), dwp=(dh * gate * u * s).sum(0))
            dg = dh * s * u * wp
            out['dgate'] = dg.sum(1, keepdim=True) if gate.shape[-1] == 1 else dg
    return out


# a row's sums of up to C terms in float32 are off by at most C 2^-24 of their magnitudes; with values of order one the
# results inherit at most that relative error, twice over (two norms), and column sums over T rows T 2^-24 of theirs
@pytest.mark.parametrize('dt', [F32, BF16, F16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('kind', ['rms', 'layer'])
@pytest.mark.parametrize('T,C,gate', [(1, 1, None), (1, 64, 'row'), (7, 129, 'full'), (160, 512, 'row'), (33, 515, 'full'),
                                      (3, 1024, None), (9, 2047, 'row'), (5, 4096, 'full'), (2, 8192, 'row'), (5000, 40, 'full')])
def test_block_norm_and_its_gradients(T, C, gate, kind, dt):
    d = dev()
    print(f'[case] block_norm T={T} C={C} gate={gate} {kind} {dt}', flush=True)
    rng = np.random.default_rng(T * 13 + C)
    eps = 1e-3 if C == 1 else 1e-6
    x, y = rand(rng, T, C, dt=dt), rand(rng, T, C, dt=dt, scale=2.0, mean=0.3)
    gt = None if gate is None else rand(rng, T, C if gate == 'full' else 1, dt=dt)
    s, wp, wn = (rand(rng, C, dt=dt, scale=0.2, mean=1.0) for _ in range(3))
    gh, gn = rand(rng, T, C, dt=dt), rand(rng, T, C, dt=dt)
    want = norm_case(x, y, gt, s, wp, wn, gh, gn, kind, eps)
    ins = [None if t is None else t.to(d).requires_grad_() for t in (x, y, gt, s, wp, wn)]
    h, n = mhk.block_norm(*ins, eps=eps, kind=kind)
    leaves = [t for t in ins if t is not None]
    grads = torch.autograd.grad((h, n), leaves, (gh.to(d), gn.to(d)), retain_graph=True)
    again = torch.autograd.grad((h, n), leaves, (gh.to(d), gn.to(d)))
    names = ['dx', 'dy'] + (['dgate'] if gate else []) + ['ds', 'dwp', 'dwn']
    for name, got, twice in zip(['h', 'n'] + names, (h, n, *grads), (h, n, *again)):
        val = want[name]
        if gate is not None and name == 'dgate':
            val = val.reshape(got.shape)
        # one channel: 'layer' gives norm(v) = 0 and 1 / sqrt(eps) times rounding differences
        # 'rms' of one channel: the derivative is eps over a cube, cancelled from order-one terms
        terms = {'ds': T, 'dwp': T, 'dwn': T, 'dgate': C}.get(name, 1)
        big = val.abs().max()
        scale = torch.maximum(val.abs(), torch.tensor(float(terms) ** 0.5 * 8 * (30.0 if C == 1 else 1.0), dtype=torch.float64))
        near(name, got, val, (C + terms + 64) * E32 * torch.maximum(scale, big) + U[dt] * val.abs() + TINY[dt])
        assert torch.equal(got, twice), f'{name} differs between two passes'
    with torch.no_grad():
        h2, n2 = mhk.block_norm(*ins, eps=eps, kind=kind)
    assert torch.equal(h, h2) and torch.equal(n, n2)


@pytest.mark.parametrize('dt', [F32, BF16], ids=['f32', 'bf16'])
def test_block_norm_without_branch_or_weights_and_partial_gradients(dt):
    d = dev()
    print(f'[case] block_norm parts {dt}', flush=True)
    rng = np.random.default_rng(6)
    T, C = 21, 96
    x, y, gn = rand(rng, T, C, dt=dt), rand(rng, T, C, dt=dt), rand(rng, T, C, dt=dt)
    wn = rand(rng, C, dt=dt)
    lx, lw = x.to(d).requires_grad_(), wn.to(d).requires_grad_()
    h, n = mhk.block_norm(lx.view(3, 7, C), pre_weight=lw)
    assert h.shape == (3, 7, C) and n.shape == (3, 7, C) and torch.equal(h.reshape(T, C), lx)
    want = norm_case(x, None, None, None, None, wn, gn, gn, 'rms', 1e-6)
    dx, dw = torch.autograd.grad(n, (lx, lw), gn.to(d).view(3, 7, C))
    tol = lambda v, k: (C + k + 64) * E32 * torch.maximum(v.abs().max(), torch.tensor(8.0)) + U[dt] * v.abs()  # noqa: E731
    near('n', n.reshape(T, C), want['n'], tol(want['n'], 1))
    near('dx', dx, want['dx'], tol(want['dx'], 1))
    near('dwn', dw, want['dwn'], tol(want['dwn'], T))
    # the stream alone used: no gradient of the normed output
    ly = y.to(d).requires_grad_()
    h, n = mhk.block_norm(x.to(d), ly)
    dy, = torch.autograd.grad(h, ly, gn.to(d))
    want = norm_case(x, y, None, None, None, None, gn, torch.zeros_like(gn), 'rms', 1e-6)
    near('dy', dy, want['dy'], tol(want['dy'], 1))
    # rows of zeros: finite, zero norms
    z = torch.zeros(4, C, dtype=dt, device=d)
    h, n = mhk.block_norm(z, z, kind='layer')
    assert (h == 0).all() and (n == 0).all()
    # a NaN row stays in its row
    bad = x.clone()
    bad[3] = float('nan')
    h, n = mhk.block_norm(bad.to(d), y.to(d))
    assert torch.isnan(n[3]).all() and torch.isfinite(n[:3].float()).all() and torch.isfinite(n[4:].float()).all()
    e = mhk.block_norm(torch.empty(0, C, dtype=dt, device=d))
    assert e[1].shape == (0, C)


# ---------------------------------------------------------------------------------------------------- all of them
def test_gradients_against_differences():
    """The gradients of a whole routed block against central differences of its own float32 forward."""
    d = dev()
    print('[case] differences', flush=True)
    torch.manual_seed(0)
    T, C, H, E, k = 12, 16, 24, 3, 2
    x0 = torch.randn(T, C, device=d)
    ps = [torch.randn(E, H, C, device=d) * 0.3, torch.randn(E, H, device=d) * 0.1, torch.randn(E, C, H, device=d) * 0.3,
          torch.rand(T, k, device=d), torch.rand(C, device=d) + 0.5, torch.rand(C, device=d) + 0.5, torch.rand(T, 1, device=d)]
    experts = torch.randint(-1, E, (T, k), device=d)
    probe = torch.randn(2, T, C, device=d)

    def loss(x, w1, b1, w2, w, post, pre, gate):
        o = mhk.expert_order(experts, E)
        _, n = mhk.block_norm(x, pre_weight=pre)
        y = mhk.expert_dense(mhk.dispatch(n, o), w1, o.offsets, b1, 'silu')
        y = mhk.combine(mhk.expert_dense(y, w2, o.offsets), w, o)
        h, n = mhk.block_norm(x, mhk.dense(y, torch.eye(C, device=d), activation='gelu'), gate=gate, post_weight=post)
        return (h * probe[0]).double().sum() + (n * probe[1]).double().sum()

    args = [t.clone().requires_grad_() for t in (x0, *ps)]
    grads = torch.autograd.grad(loss(*args), args)
    step = 2.0 ** -7
    for i, g in enumerate(grads):
        v = torch.randn_like(args[i])
        v /= v.norm()
        with torch.no_grad():
            f = [float(loss(*(a + s * step * v if j == i else a for j, a in enumerate(args)))) for s in (1, -1, 2, -2)]
        # fourth-order differences: the error of f is about 2^-22 of sums of a few hundred, over the step
        num = (8 * (f[0] - f[1]) - (f[2] - f[3])) / (12 * step)
        ana = float((g.double() * v.double()).sum())
        assert abs(num - ana) < 2e-2 * max(1.0, abs(ana)), (i, num, ana)


def test_another_stream_and_a_captured_graph():
    d = dev()
    print('[case] streams and graphs', flush=True)
    torch.manual_seed(1)
    x, w = torch.randn(300, 64, device=d), torch.randn(4, 64, 64, device=d)
    experts = torch.randint(0, 4, (300, 2), device=d)
    gate = torch.rand(300, 2, device=d)

    def call():
        o = mhk.expert_order(experts, 4)
        _, n = mhk.block_norm(x)
        y = mhk.combine(mhk.expert_dense(mhk.dispatch(n, o), w, o.offsets, activation='silu'), gate, o, residual=x)
        return mhk.dense(y, w[0], activation='gelu')

    want = call()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = call()
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(3):
        with torch.no_grad():
            x.normal_()
            experts.random_(-1, 4)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call()), i


def test_double_backward_raises():
    d = dev()
    x = torch.randn(4, 8, device=d, requires_grad=True)
    o = mhk.expert_order(torch.zeros(4, 1, dtype=torch.int64, device=d), 1)
    for f in (lambda: mhk.dense(x, torch.eye(8, device=d), activation='silu'), lambda: mhk.block_norm(x)[1],
              lambda: mhk.dispatch(x, o), lambda: mhk.combine(x, None, o)):
        with pytest.raises(RuntimeError, match='double backward'):
            torch.autograd.grad(f().sum(), x, create_graph=True)


def test_refusals_on_the_gpu():
    d = dev()
    x, w = torch.zeros(4, 8, device=d), torch.zeros(6, 8, device=d)
    o = mhk.expert_order(torch.zeros(4, 2, dtype=torch.int32, device=d), 3)
    off = torch.zeros(4, dtype=torch.int32, device=d)
    for call, kind, text in [
            (lambda: mhk.dense(x, w.bfloat16()), TypeError, 'weight must be'),
            (lambda: mhk.dense(x, w.cpu()), TypeError, 'weight must be'),
            (lambda: mhk.dense(x, torch.zeros(6, 9, device=d)), ValueError, 'weight must be'),
            (lambda: mhk.dense(x, torch.zeros(2, 6, 8, device=d)), ValueError, 'weight must be'),
            (lambda: mhk.dense(x, w, torch.zeros(5, device=d)), ValueError, 'bias must be'),
            (lambda: mhk.dense(x, w, residual=x), ValueError, 'residual must be'),
            (lambda: mhk.dense(x, w, activation='tanh'), ValueError, 'activation must be'),
            (lambda: mhk.dense(x.double(), w.double()), TypeError, 'float32, bfloat16 or float16'),
            (lambda: mhk.expert_dense(x, torch.zeros(3, 6, 8, device=d), off.long()), TypeError, 'offsets must be'),
            (lambda: mhk.expert_dense(x, torch.zeros(3, 6, 8, device=d), off[:3]), ValueError, 'offsets must be'),
            (lambda: mhk.expert_dense(x[None], torch.zeros(3, 6, 8, device=d), off), ValueError, 'rows'),
            (lambda: mhk.expert_order(x, 3), TypeError, 'int32 or int64'),
            (lambda: mhk.expert_order(o.place[0], 3), ValueError, r'\[T, k\]'),
            (lambda: mhk.expert_order(o.place, 0), ValueError, 'n_experts'),
            (lambda: mhk.expert_order(o.place, 1025), ValueError, 'n_experts'),
            (lambda: mhk.dispatch(x[:3], o), ValueError, 'x must be'),
            (lambda: mhk.dispatch(x, o.place), TypeError, 'expert_order'),
            (lambda: mhk.combine(x, None, o), ValueError, 'y must be'),
            (lambda: mhk.combine(torch.zeros(8, 3, device=d), torch.zeros(4, 1, device=d), o), ValueError, 'weights must be'),
            (lambda: mhk.combine(torch.zeros(8, 3, device=d), torch.zeros(4, 2, device=d).half(), o), TypeError, 'weights must'),
            (lambda: mhk.block_norm(x, gate=x), ValueError, 'belong to a branch'),
            (lambda: mhk.block_norm(x, x, gate=x[:, :2]), ValueError, 'gate must be'),
            (lambda: mhk.block_norm(x, x[:2]), ValueError, 'y must be'),
            (lambda: mhk.block_norm(x, kind='batch'), ValueError, 'kind must be'),
            (lambda: mhk.block_norm(x, eps=-1.0), ValueError, 'eps'),
            (lambda: mhk.block_norm(torch.zeros(2, norms.MAX_CHANNELS + 1, device=d)), ValueError, 'channels')]:
        with pytest.raises(kind, match=text):
            call()
    assert set(matmul.TYPES) == {F32, BF16, F16}


@pytest.mark.parametrize('dt', [F32, BF16], ids=['f32', 'bf16'])
def test_gradients_at_odd_places(dt):
    """A gradient in rows of a wider tensor, off the steps of 16 bytes that its width promises, against the same copied."""
    d = dev()
    rng = np.random.default_rng(77)
    x, w, b = (rand(rng, *s, dt=dt).to(d).requires_grad_() for s in ((300, 64), (72, 64), (72,)))
    wide = rand(rng, 300, 83, dt=dt).to(d)
    for act in (None, 'silu'):
        y = mhk.dense(x, w, b, act)
        for g in (wide[:, 3:75], wide[:, :72]):
            print(f'[case] gradient at odd places {dt} {act}', flush=True)
            a = torch.autograd.grad(y, (x, w, b), g, retain_graph=True)
            c = torch.autograd.grad(y, (x, w, b), g.contiguous(), retain_graph=True)
            for name, s, t in zip(('dx', 'dw', 'db'), a, c):
                r = (s.double() - t.double()).norm() / t.double().norm()
                assert r <= 8 * {F32: 2 ** -24, BF16: 2 ** -8}[dt], (name, act, float(r))


def test_launches_are_timed_in_both_directions():
    d = dev()
    x, w = torch.randn(40, 32, device=d, requires_grad=True), torch.randn(24, 32, device=d, requires_grad=True)
    with _native.timing() as tm:
        mhk.block_norm(mhk.dense(x, w))[1].sum().backward()
    seen = tm.summary()
    assert {'mm_fwd', 'nm_fwd', 'nm_bwd', 'mm_bwd'} <= set(seen), seen
    assert 'mm_fwd' in tm.symbols['mm_fwd'] and 'mm_dx' in tm.symbols['mm_bwd'], tm.symbols
    n = len(tm.records)
    mhk.dense(x, w).sum().backward()
    assert len(tm.records) == n


def test_a_tensor_that_changed_its_shape_is_refused():
    d = dev()
    x, w = torch.randn(40, 32, device=d, requires_grad=True), torch.randn(24, 32, device=d, requires_grad=True)
    y = mhk.dense(x, w)
    x.data = torch.randn(8, 32, device=d)
    with pytest.raises(RuntimeError, match='changed its shape|Expected'):
        y.sum().backward()


@pytest.mark.parametrize('dt', [F32, BF16, F16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('N', [64, 51])
def test_slopes_of_nan_stay_in_their_rows(N, dt):
    """A NaN input makes its own row's output and gradient NaN, the others keep the values they have without it."""
    d = dev()
    rng = np.random.default_rng(N)
    x, w, g = rand(rng, 70, 40, dt=dt).to(d), rand(rng, N, 40, dt=dt).to(d), rand(rng, 70, N, dt=dt).to(d)
    bad = x.clone()
    bad[3, 7] = float('nan')
    for act in ('silu', 'gelu'):
        print(f'[case] NaN slopes {dt} N={N} {act}', flush=True)
        (y, dx), (z, dz) = ((o, torch.autograd.grad(o, i, g)[0]) for i in (x.clone().requires_grad_(), bad.clone().requires_grad_())
                            for o in (mhk.dense(i, w, None, act),))
        keep = torch.arange(70, device=d) != 3
        assert z[3].isnan().all() and dz[3].isnan().all(), act
        assert torch.equal(y[keep], z[keep]) and torch.equal(dx[keep], dz[keep]) and dx.isfinite().all(), act


@pytest.mark.parametrize('dt', [F32, BF16, F16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('kind', ['rms', 'layer'])
@pytest.mark.parametrize('T,C,gate', [(1, 2, 'row'), (65, 16, 'full'), (130, 33, None), (77, 100, 'row'), (1000, 130, 'full'),
                                      (200, 255, 'row'), (2100, 257, None)])
def test_block_norm_of_narrow_rows(T, C, gate, kind, dt):
    """Rows that several to a wave are taken: T that fills no workgroup, C on both sides of each split."""
    test_block_norm_and_its_gradients(T, C, gate, kind, dt)
