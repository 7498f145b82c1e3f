"""
Trains a head on the node features of a patched model: the backbone runs on the HIP drop-ins (its weights are constants
there), the head's layers are the trainable ones (dense, expert_dense, expert_order, dispatch, combine, block_norm).

    python examples/train_node_head.py [--steps 60] [--dtype float32|bfloat16|float16] [--router]

Structures are seeded Pt slabs with C/O/H adsorbates; the per-atom target is a smooth function of each atom's own neighbour
distances with a strength per element, so that a head with an expert per element has something to learn.
"""
import argparse
import os
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (os.path.join(ROOT, 'mace-mps-kernels_amd'), ROOT):
    if p not in sys.path:
        sys.path.insert(0, p)

from mace_hip_kernels import NodeHead, node_features, patch_model  # noqa: E402
from mace_lite import data as D  # noqa: E402
from mace_lite import factory  # noqa: E402


def dataset(device, slabs=6, seed=0):
    """(node features [N, C], element index [N], target [N]) of a batch of slabs."""
    rng = np.random.default_rng(seed)
    elements = factory.ELEMENTS_PTCOH
    structures = [factory.pt_slab_with_adsorbates(rng, (4, 4, 4), 15) for _ in range(slabs)]
    batch = D.batch_graphs([D.graph_of(s, 5.0) for s in structures], elements, device=device)
    model = factory.make_model('32x0e+32x1o', 2, 2, elements=elements).to(device).eval()
    for p in model.parameters():
        p.requires_grad_(False)
    patch_model(model, verbose=False)
    feats = node_features(model, D.fresh(batch))[:, :32]
    kind = batch['node_attrs'].detach().argmax(1)
    send, recv = batch['edge_index']
    pos = batch['positions'].detach()
    vec = pos[recv] - pos[send] + batch['shifts']
    pair = torch.exp(-vec.norm(dim=1))
    strength = torch.tensor([1.0, -2.0, 1.5, 0.5], device=device)
    target = torch.zeros(len(kind), device=device).index_add_(0, recv, pair) * strength[kind]
    return (feats - feats.mean(0)) / (feats.std(0) + 1e-6), kind, (target - target.mean()) / target.std()


def train(steps=60, dtype=torch.float32, router=False, seed=0, device='cuda'):
    """The mean squared errors of the steps."""
    torch.manual_seed(seed)
    feats, kind, target = dataset(torch.device(device))
    head = NodeHead(feats.shape[1], 64, hidden=128, layers=2, n_experts=4, top_k=2 if router else 0, dtype=dtype).to(device)
    opt = torch.optim.Adam(head.parameters(), lr=3e-3)
    losses = []
    for _ in range(steps):
        opt.zero_grad(set_to_none=True)
        loss = (head(feats, None if router else kind) - target).square().mean()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument('--steps', type=int, default=60)
    ap.add_argument('--dtype', choices=('float32', 'bfloat16', 'float16'), default='float32')
    ap.add_argument('--router', action='store_true', help='experts chosen by a learned router, two per node')
    a = ap.parse_args()
    losses = train(a.steps, getattr(torch, a.dtype), a.router)
    for i in sorted({0, len(losses) // 4, len(losses) // 2, len(losses) - 1}):
        print(f'step {i:4d}  mean squared error {losses[i]:.4f}', flush=True)


if __name__ == '__main__':
    main()
