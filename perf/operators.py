"""
The trainable layers on a backbone's node features, as cases that can be timed: the matrix product with its epilogue
(``dense``), the experts' products over groups of rows (``expert_dense``), the rows sorted by expert and back
(``expert_order``, ``dispatch``, ``combine``) and the norms around a block (``block_norm``), forward alone (answering) or
with all gradients (training).

A case is a dict of plain values.  ``prepare`` makes the inputs, ``run`` is one pass: by the framework's operators where
``own`` is true, else in elementary torch operations in 32 bits, rounded once at the end.  ``exact`` is the same in 64.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
_EPS = 1e-6


def _hip():
    """The framework's package, imported where its operators are called."""
    mod = sys.modules.get('mace_hip_kernels')
    if mod is None:
        path = os.path.abspath('mace-mps-kernels_amd')
        if path not in sys.path:
            sys.path.insert(0, path)
        import mace_hip_kernels as mod
    return mod


# --------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one node through a wide layer: the call of a single query, bound by its latency and the weights' bytes
        dict(name='dense_one', op='dense', T=1, K=1024, N=4096, act='silu', res=False, train=False, dtype='bfloat16'),
        # the atoms of sixteen slabs through the first layer of a feed-forward block on 128 channels, trained
        dict(name='dense_slabs16', op='dense', T=2533, K=128, N=512, act='silu', res=False, train=True, dtype='float32'),
        # sizes that no tile divides: concatenated descriptors of odd lengths
        dict(name='dense_odd', op='dense', T=1999, K=515, N=1021, act='gelu', res=True, train=False, dtype='float16'),
        # a square layer with its skip connection over the atoms of a large crystal
        dict(name='dense_bulk20000', op='dense', T=20000, K=1024, N=1024, act='none', res=True, train=False, dtype='float32'),
        # one training step of the wide layer of a large model over a batch of 16,384 nodes
        dict(name='dense_train', op='dense', T=16384, K=1024, N=4096, act='silu', res=False, train=True, dtype='bfloat16'),
        # four nodes, two experts each of sixty-four: the weights of the few experts met are what is read
        dict(name='experts_few', op='experts', R=8, E=64, K=1024, N=2048, act='silu', res=False, train=False, dtype='bfloat16'),
        # per-element layers of four elements of which one is most of the crystal, answering
        dict(name='experts_elements', op='experts', R=20000, E=4, K=128, N=512, act='silu', res=False, train=False, dtype='float32'),
        # a training step of eight experts over 8,192 nodes, two each
        dict(name='experts_train', op='experts', R=16384, E=8, K=1024, N=2048, act='silu', res=False, train=True, dtype='bfloat16'),
        # one slab's atoms to one expert each and back
        dict(name='route_slab', op='route', T=160, k=1, E=4, C=128, train=False, dtype='float32'),
        # a training step's rows: four of 128 experts each, some dropped by their experts' capacity
        dict(name='route_train', op='route', T=32768, k=4, E=128, C=1024, train=True, dtype='bfloat16'),
        # the norms of one slab's atoms, answering
        dict(name='norm_slab', op='norm', T=160, C=512, kind='rms', gate='row', train=False, dtype='bfloat16'),
        # the norms of a large batch, trained, with a gate of its own for each channel
        dict(name='norm_train', op='norm', T=32768, C=2048, kind='rms', gate='full', train=True, dtype='bfloat16'),
    ]


def _log(rng, lo, hi):
    """Spread over the logarithm; half of the values multiples of eight where there is room."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v >= 32 and rng.random() < 0.5:
        v = v // 8 * 8
    return v if v != 3072 else 3080


def draw(rng):
    most = {c['name']: _cost(c) for c in listed()}
    cap = {'dense': most['dense_train'], 'experts': most['experts_train'], 'route': most['route_train'],
           'norm': most['norm_train']}
    while True:
        op = rng.choice(['dense', 'dense', 'experts', 'route', 'norm'])
        c = dict(op=op, train=rng.random() < 0.5, dtype=rng.choice(['float32', 'bfloat16', 'float16']))
        if op == 'dense':
            c.update(T=_log(rng, 1, 20000), K=_log(rng, 16, 2048), N=_log(rng, 16, 4096),
                     act=rng.choice(['none', 'relu', 'silu', 'gelu']), res=rng.random() < 0.5)
        elif op == 'experts':
            c.update(R=_log(rng, 1, 20000), E=_log(rng, 1, 128), K=_log(rng, 16, 2048), N=_log(rng, 16, 2048),
                     act=rng.choice(['none', 'silu', 'gelu']), res=rng.random() < 0.3)
            if c['E'] * c['K'] * c['N'] > 2 ** 28:
                continue
        elif op == 'route':
            c.update(T=_log(rng, 1, 32768), k=rng.randint(1, 4), E=_log(rng, 4, 128), C=_log(rng, 16, 2048))
        else:
            c.update(T=_log(rng, 1, 32768), C=_log(rng, 16, 4096), kind=rng.choice(['rms', 'layer']),
                     gate=rng.choice(['none', 'row', 'full']))
        if _cost(c) <= cap[op]:
            return c


def _cost(c):
    w = work(c)
    return max(w['bytes'], w['flops'] / 50)


def work(c):
    """Bytes and operations of one pass: every input read once, every output written once."""
    s = 4 if c['dtype'] == 'float32' else 2
    if c['op'] == 'norm':
        T, C = c['T'], c['C']
        gate = {'none': 0, 'row': T, 'full': T * C}[c['gate']]
        if not c['train']:
            return dict(bytes=s * (4 * T * C + gate + 3 * C), flops=12 * T * C)
        return dict(bytes=s * (8 * T * C + 2 * gate + 6 * C), flops=42 * T * C)
    if c['op'] == 'route':
        T, k, E, C = c['T'], c['k'], c['E'], c['C']
        A = T * k
        order = 4 * (A + 2 * A + E + 1)
        fwd = s * (T * C + A * C) + s * (A * C + T * C) + 4 * A
        bwd = s * (A * C + T * C) + s * (T * C + A * C) + 4 * A
        return dict(bytes=order + fwd + (bwd if c['train'] else 0), flops=(2 + (4 if c['train'] else 0)) * A * C)
    T, K, N = c.get('T', c.get('R')), c['K'], c['N']
    E = min(c.get('E', 1), T)                                   # experts that can have a row
    fwd = s * (T * K + E * N * K + E * N + T * N * (2 if c['res'] else 1))
    flops = 2 * T * N * K
    if not c['train']:
        return dict(bytes=fwd, flops=flops)
    return dict(bytes=fwd + s * (T * N + T * K + c.get('E', 1) * N * (K + 1)), flops=3 * flops)


# -------------------------------------------------------------------------------------------------------- inputs
def _inputs(c, seed):
    dev = torch.device('cuda', torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    dt = _DTYPES[c['dtype']]

    def normal(*shape, scale=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale + mean).to(dt)

    s = {}
    if c['op'] == 'norm':
        T, C = c['T'], c['C']
        s.update(x=normal(T, C), y=normal(T, C, scale=2.0, mean=0.1), wp=normal(C, scale=0.1, mean=1.0),
                 wn=normal(C, scale=0.1, mean=1.0), scale=normal(C, scale=0.1, mean=0.5))
        if c['gate'] != 'none':
            s['gate'] = normal(T, C if c['gate'] == 'full' else 1, scale=0.3, mean=0.5)
        if c['train']:
            s.update(gh=normal(T, C), gn=normal(T, C))
        return s
    if c['op'] == 'route':
        T, k, E, C = c['T'], c['k'], c['E'], c['C']
        # distinct experts of each node by noisy scores with a preference among the experts, 3% dropped
        score = -torch.log(-torch.log(torch.rand(T, E, generator=g, device=dev).clamp(1e-7, 1 - 1e-7)))
        score = score + torch.linspace(0, 1.5, E, device=dev)
        top = torch.topk(score, k, dim=1)
        keep = torch.rand(T, k, generator=g, device=dev) >= 0.03
        s.update(experts=torch.where(keep, top.indices, -1).to(torch.int32), w=torch.softmax(top.values, dim=1),
                 x=normal(T, C), y=normal(T * k, C))
        if c['train']:
            s.update(gx=normal(T * k, C), go=normal(T, C))
        return s
    T, K, N = c.get('T', c.get('R')), c['K'], c['N']
    lead = (c['E'],) if c['op'] == 'experts' else ()
    s.update(x=normal(T, K), w=normal(*lead, N, K, scale=K ** -0.5), b=normal(*lead, N, scale=0.1))
    if c['res']:
        s['r'] = normal(T, N)
    if c['train']:
        s['g'] = normal(T, N)
    if lead:
        # group sizes by a preference among the experts; the first expert (of several) has no row
        E = c['E']
        p = torch.exp(torch.linspace(0, 1.5, E, device=dev) * (2.0 if E <= 8 else 1.0))
        if E > 1:
            p[0] = 0
        e = torch.multinomial(p, T, replacement=True, generator=g)
        s['offsets'] = torch.searchsorted(torch.sort(e).values, torch.arange(E + 1, device=dev)).to(torch.int32)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case['op'] == 'experts':
        # the plain form lays the groups out at one length each: the largest, which a program knows from its counts
        s['longest'] = int((s['offsets'][1:] - s['offsets'][:-1]).max())
    s['case'] = case
    return s


# ------------------------------------------------------------------------------------------------- one pass, plain
def _act(name, a):
    if name == 'relu':
        return a.clamp_min(0)
    if name == 'silu':
        return a / (1 + torch.exp(-a))
    if name == 'gelu':
        return 0.5 * a * (1 + torch.erf(a * 0.5 ** 0.5))
    return a


def _act_slope(name, a):
    if name == 'relu':
        return (a > 0).to(a.dtype)
    if name == 'silu':
        q = 1 / (1 + torch.exp(-a))
        return q * (1 + a * (1 - q))
    return 0.5 * (1 + torch.erf(a * 0.5 ** 0.5)) + a * torch.exp(-0.5 * a * a) * (2 * math.pi) ** -0.5


def _plain_dense(s, c):
    dt = s['x'].dtype
    x, w = s['x'].float(), s['w'].float()
    a = x @ w.t() + s['b'].float()
    y = _act(c['act'], a)
    if c['res']:
        y = y + s['r'].float()
    out = dict(y=y.to(dt))
    if c['train']:
        p = s['g'].float()
        if c['act'] != 'none':
            p = p * _act_slope(c['act'], a)
        out.update(dx=(p @ w).to(dt), dw=(p.t() @ x).to(dt), db=p.sum(0).to(dt))
    return out


def _plain_experts(s, c):
    dt, E, R = s['x'].dtype, c['E'], c['R']
    x, b, off = s['x'].float(), s['b'].float(), s['offsets'].long()
    e = torch.searchsorted(off, torch.arange(R, device=x.device), right=True) - 1         # the row's expert
    if R <= E and not c['train']:
        a = torch.bmm(s['w'][e].float(), x[:, :, None])[:, :, 0] + b[e]                  # a row each
        y = _act(c['act'], a)
        return dict(y=(y + s['r'].float() if c['res'] else y).to(dt))
    w, n = s['w'].float(), s['longest']
    at = e * n + torch.arange(R, device=x.device) - off[e]                               # the row's place among them

    def spread(v):
        return v.new_zeros(E * n, v.shape[1]).index_copy_(0, at, v).view(E, n, -1)

    xs = spread(x)
    a = torch.bmm(xs, w.transpose(1, 2).contiguous()).view(E * n, -1)[at] + b[e]
    y = _act(c['act'], a)
    out = dict(y=(y + s['r'].float() if c['res'] else y).to(dt))
    if c['train']:
        p = s['g'].float()
        if c['act'] != 'none':
            p = p * _act_slope(c['act'], a)
        ps = spread(p)
        out.update(dx=torch.bmm(ps, w).view(E * n, -1)[at].to(dt), db=ps.sum(1).to(dt),
                   dw=torch.bmm(ps.transpose(1, 2).contiguous(), xs).to(dt))
    return out


def _plain_route(s, c):
    T, k, E, dt = c['T'], c['k'], c['E'], s['x'].dtype
    flat = s['experts'].reshape(-1).long()
    kept = flat >= 0
    key = torch.where(kept, flat, E)
    order = torch.argsort(key, stable=True)
    offsets = torch.searchsorted(key[order], torch.arange(E + 1, device=flat.device))
    here = torch.arange(T * k, device=flat.device) < offsets[-1]                          # places that have a row
    rows = torch.where(here, order, -1)
    place = torch.empty_like(order).index_copy_(0, order, torch.arange(T * k, device=flat.device))
    xs = s['x'][order // k] * here[:, None]
    w = torch.where(kept, s['w'].reshape(-1), 0.0)
    y = s['y'].float()[place].view(T, k, -1)
    out = dict(offsets=offsets.int(), rows=rows.int(), place=torch.where(kept, place, -1).int().view(T, k), xs=xs,
               out=(y * w.view(T, k, 1)).sum(1).to(dt))
    if c['train']:
        go = s['go'].float()
        out.update(dx=(s['gx'].float()[place] * kept[:, None]).view(T, k, -1).sum(1).to(dt),
                   dy=(go[order // k] * (w[order] * here)[:, None]).to(dt),
                   dw=((y * go[:, None]).sum(2) * kept.view(T, k)))
    return out


def _plain_norm(s, c):
    dt = s['x'].dtype
    x, y, wp, wn, sc = (s[k].float() for k in ('x', 'y', 'wp', 'wn', 'scale'))
    gate = s['gate'].float() if 'gate' in s else x.new_ones(1, 1)

    def norm(v):
        if c['kind'] == 'layer':
            v = v - v.mean(1, keepdim=True)
        r = 1 / torch.sqrt((v * v).mean(1, keepdim=True) + _EPS)
        return v * r, r

    def back(g, v, r):
        d = g - v * (g * v).mean(1, keepdim=True)
        if c['kind'] == 'layer':
            d = d - g.mean(1, keepdim=True)
        return d * r

    u, ru = norm(y)
    h = x + sc * gate * (u * wp)
    v, rv = norm(h)
    out = dict(h=h.to(dt), n=(v * wn).to(dt))
    if c['train']:
        gn = s['gn'].float()
        dh = s['gh'].float() + back(gn * wn, v, rv)
        out.update(dx=dh.to(dt), dwn=(gn * v).sum(0).to(dt), dscale=(dh * gate * u * wp).sum(0).to(dt),
                   dwp=(dh * gate * u * sc).sum(0).to(dt), dy=back(dh * gate * sc * wp, u, ru).to(dt))
        if 'gate' in s:
            dg = dh * sc * u * wp
            out['dgate'] = (dg.sum(1, keepdim=True) if c['gate'] == 'row' else dg).to(dt)
    return out


# ------------------------------------------------------------------------------------ one pass, by the framework
def _grads(names, ins, outs, seeds):
    return dict(zip(names, torch.autograd.grad(outs, ins, seeds)))


def _leaves(s, *names):
    return [s[n].detach().requires_grad_() for n in names]


def _own(s, c):
    mhk, train = _hip(), c['train']
    if c['op'] == 'norm':
        names = ['x', 'y', 'wp', 'wn', 'scale'] + (['gate'] if 'gate' in s else [])
        v = dict(zip(names, _leaves(s, *names))) if train else s
        h, n = mhk.block_norm(v['x'], v['y'], gate=v.get('gate'), scale=v['scale'], post_weight=v['wp'],
                              pre_weight=v['wn'], eps=_EPS, kind=c['kind'])
        out = dict(h=h.detach(), n=n.detach())
        if train:
            out.update(_grads(['d' + k for k in names], [v[k] for k in names], (h, n), (s['gh'], s['gn'])))
        return out
    if c['op'] == 'route':
        v = dict(zip('xyw', _leaves(s, 'x', 'y', 'w'))) if train else s
        order = mhk.expert_order(s['experts'], c['E'])
        xs = mhk.dispatch(v['x'], order)
        y = mhk.combine(v['y'], v['w'], order)
        out = dict(offsets=order.offsets, rows=order.rows, place=order.place, xs=xs.detach(), out=y.detach())
        if train:
            out.update(_grads(['dx', 'dy', 'dw'], [v['x'], v['y'], v['w']], (xs, y), (s['gx'], s['go'])))
        return out
    v = dict(zip('xwb', _leaves(s, 'x', 'w', 'b'))) if train else s
    res, act = s.get('r'), None if c['act'] == 'none' else c['act']
    if c['op'] == 'dense':
        y = mhk.dense(v['x'], v['w'], bias=v['b'], activation=act, residual=res)
    else:
        y = mhk.expert_dense(v['x'], v['w'], s['offsets'], bias=v['b'], activation=act, residual=res)
    out = dict(y=y.detach())
    if train:
        out.update(_grads(['dx', 'dw', 'db'], [v['x'], v['w'], v['b']], (y,), (s['g'],)))
    return out


def run(state):
    c = state['case']
    if own:
        return _own(state, c)
    return {'dense': _plain_dense, 'experts': _plain_experts, 'route': _plain_route, 'norm': _plain_norm}[c['op']](state, c)


# ----------------------------------------------------------------------------------------------- the same in 64 bits
def _ddense(x, w, b, act, r, g):
    """y and the gradients by x, w and b of act(x w^T + b) + r for the gradient g of y, in float64 by autograd."""
    x, w, b = (t.detach().requires_grad_() for t in (x, w, b))
    f = {'none': lambda a: a, 'relu': torch.relu, 'silu': torch.nn.functional.silu, 'gelu': torch.nn.functional.gelu}[act]
    y = f(torch.addmm(b, x, w.t()))
    if r is not None:
        y = y + r
    if g is None:
        return dict(y=y.detach())
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
    return dict(y=y.detach(), dx=dx, dw=dw, db=db)


def exact(case, seed):
    c = case
    s = {k: v.double() if v.is_floating_point() else v for k, v in _inputs(c, seed).items()}
    if c['op'] == 'dense':
        return _ddense(s['x'], s['w'], s['b'], c['act'], s.get('r'), s.get('g'))
    if c['op'] == 'experts':
        off = s['offsets'].tolist()
        parts = []
        for e in range(c['E']):
            i = slice(off[e], off[e + 1])
            parts.append(_ddense(s['x'][i], s['w'][e], s['b'][e], c['act'], s['r'][i] if c['res'] else None,
                                 s['g'][i] if c['train'] else None))
        return {k: (torch.stack if k in ('dw', 'db') else torch.cat)([p[k] for p in parts]) for k in parts[0]}
    if c['op'] == 'route':
        T, k, E, C = c['T'], c['k'], c['E'], c['C']
        flat = s['experts'].reshape(-1).tolist()
        lists = [[] for _ in range(E)]
        for i, e in enumerate(flat):
            if e >= 0:
                lists[e].append(i)
        at = torch.tensor([i for li in lists for i in li], dtype=torch.long, device=s['x'].device)    # place -> flat
        n, A = at.numel(), T * k
        token = at // k
        w = s['w'].reshape(-1)[at]
        zeros = s['x'].new_zeros
        out = dict(offsets=None, rows=None, place=None, xs=torch.cat([s['x'][token], zeros(A - n, C)]),
                   out=zeros(T, C).index_add_(0, token, s['y'][:n] * w[:, None]))
        if c['train']:
            go = s['go'][token]
            out.update(dx=zeros(T, C).index_add_(0, token, s['gx'][:n]), dy=torch.cat([go * w[:, None], zeros(A - n, C)]),
                       dw=zeros(A).index_add_(0, at, (go * s['y'][:n]).sum(1)).view(T, k))
        return out
    names = ['x', 'y', 'wp', 'wn', 'scale'] + (['gate'] if 'gate' in s else [])
    v = {n: s[n].detach().requires_grad_(c['train']) for n in names}

    def norm(t, w):
        if c['kind'] == 'layer':
            return torch.nn.functional.layer_norm(t, (t.shape[1],), w, None, _EPS)
        return t * torch.rsqrt(t.square().mean(1, keepdim=True) + _EPS) * w

    h = v['x'] + v['scale'] * (v['gate'] if 'gate' in v else 1.0) * norm(v['y'], v['wp'])
    n = norm(h, v['wn'])
    out = dict(h=h.detach(), n=n.detach())
    if c['train']:
        out.update(_grads(['d' + k for k in names], [v[k] for k in names], (h, n), (s['gh'], s['gn'])))
    return out
