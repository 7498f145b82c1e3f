"""
NodeFeedForward and NodeHead (every trainable node layer together) against the same formulas in float64, and the example
that trains a head on a patched model's node features.
"""
import os
import sys

import pytest
import torch

import mace_hip_kernels as mhk

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu


def plain(head, feats, experts):
    """The head's output in float64 on the CPU by torch expressions, with its parameters as leaves (named as its own)."""
    P = {k: v.detach().double().cpu().requires_grad_() for k, v in head.named_parameters()}

    def norm(v, w):
        return v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-6) * w

    h = feats.double().cpu() @ P['embed'].t()
    n = norm(h, P['pre_weight'])
    for i in range(len(head.blocks)):
        p = {k.split('.', 2)[2]: v for k, v in P.items() if k.startswith(f'blocks.{i}.')}
        if head.top_k:
            w, e = torch.topk(torch.softmax(n @ P[f'routers.{i}'].t(), 1), head.top_k, dim=1)
        elif experts is not None:
            e = experts.cpu().reshape(len(n), -1)
            w = torch.ones(e.shape, dtype=torch.float64)
        if head.n_experts:
            y = torch.zeros_like(h)
            for j in range(e.shape[1]):
                for x in range(head.n_experts):
                    sel = (e[:, j] == x).nonzero()[:, 0]
                    a = torch.nn.functional.silu(n[sel] @ p['w1'][x].t() + p['b1'][x])
                    y = y.index_add(0, sel, (a @ p['w2'][x].t() + p['b2'][x]) * w[sel, j:j + 1])
        else:
            y = torch.nn.functional.silu(n @ p['w1'].t() + p['b1']) @ p['w2'].t() + p['b2']
        g = torch.sigmoid(n @ p['wg'].t() + p['bg'])
        h = h + p['scale'] * g * norm(y, p['post_weight'])
        n = norm(h, p['pre_weight'])
    return (n @ P['readout'].t())[:, 0], P


# float32: sums of up to 256 terms in a dozen layers, 2^-24 each, amplified by the norms' divisions: 1e-4 of the largest value
@pytest.mark.parametrize('experts,top_k', [(0, 0), (4, 0), (5, 2)], ids=['shared', 'given', 'router'])
@pytest.mark.parametrize('n', [1, 60, 700])
def test_head_matches_float64(n, experts, top_k):
    print(f'[case] head n={n} experts={experts} top_k={top_k}', flush=True)
    torch.manual_seed(3)
    head = mhk.NodeHead(24, 64, hidden=96, layers=2, n_experts=experts, top_k=top_k).cuda()
    feats = torch.randn(n, 24, device='cuda')
    e = torch.randint(-1, experts, (n,), device='cuda') if experts and not top_k else None
    out = head(feats, e)
    want, P = plain(head, feats, e)
    g = torch.randn(n, dtype=torch.float64)
    out.backward(g.float().cuda())
    grads = torch.autograd.grad(want, list(P.values()), g, allow_unused=True)
    assert out.shape == (n,) and (out.double().cpu() - want).abs().max() <= 1e-4 * want.abs().max().clamp_min(1)
    for (name, p), w in zip(head.named_parameters(), grads):
        w = torch.zeros(p.shape, dtype=torch.float64) if w is None else w
        got = torch.zeros_like(w) if p.grad is None else p.grad.double().cpu()
        assert (got - w).abs().max() <= 1e-4 * max(1.0, float(w.abs().max())), name


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_head_in_16_bits_follows_float32(dtype):
    print(f'[case] head in {dtype}', flush=True)
    torch.manual_seed(4)
    head = mhk.NodeHead(32, 64, layers=1, n_experts=4, dtype=dtype).cuda()
    feats, e = torch.randn(500, 32, device='cuda'), torch.randint(0, 4, (500,), device='cuda')
    low = head(feats, e)
    head.dtype = torch.float32
    full = head(feats, e)
    # a dozen roundings of 2^-8 (2^-11) of values of order one
    assert (low - full).abs().max() < 12 * (2 ** -8 if dtype == torch.bfloat16 else 2 ** -11) * full.abs().max()


@pytest.mark.parametrize('router', [False, True])
def test_example_trains_a_head_on_a_patched_model(router):
    print(f'[case] example, router={router}', flush=True)
    sys.path.insert(0, os.path.join(ROOT, 'examples'))
    try:
        from train_node_head import train
    finally:
        sys.path.pop(0)
    losses = train(steps=60, router=router)
    assert losses[0] > 0.5 and losses[-1] < 0.2 * losses[0], losses[::10]


def test_head_refusals():
    with pytest.raises(ValueError, match='top_k'):
        mhk.NodeHead(8, 16, n_experts=2, top_k=3)
    head = mhk.NodeHead(8, 16, n_experts=2).cuda()
    with pytest.raises(ValueError, match='experts'):
        head(torch.zeros(3, 8, device='cuda'))
