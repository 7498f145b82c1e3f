"""
Trainable layers on a backbone's invariant node features, built from ``dense``, ``expert_dense``, ``expert_order``,
``dispatch``, ``combine`` and ``block_norm``: ``NodeFeedForward``, a block between its two norms, and ``NodeHead``, a stack
of them from node features to one value per node.  A patched backbone holds its weights as constants; a head is what a user
trains on the features it gives:

    feats = node_features(model, batch)[:, :128]                       # invariant channels, no gradient
    head = NodeHead(128, 256, hidden=1024, layers=2, n_experts=4).cuda()
    energy = head(feats, elements)                                     # [N]; elements [N]: each node's expert
    loss(energy).backward()

Parameters are float32; ``dtype`` is what the layers compute in.  The reference has no such layers.
"""
import torch

from .experts import combine, dispatch, expert_order
from .matmul import dense, expert_dense
from .norms import block_norm


def _weight(*shape):
    """A layer's weight, normal with variance 1 / its inputs."""
    return torch.nn.Parameter(torch.randn(shape) * shape[-1] ** -0.5)


class NodeFeedForward(torch.nn.Module):
    """h = x + scale gate norm(f(n)) post_weight and the next block's input norm(h) pre_weight, for a node's stream x and its
    normed input n: f two layers of ``hidden`` units, shared by all nodes (n_experts 0) or one of n_experts; gate =
    sigmoid of a learned projection of n, one value a node.  ``forward(x, n, experts, weights)`` takes experts [N, k] and
    their weights [N, k] (None: 1)."""

    def __init__(self, channels, hidden, n_experts=0, activation='silu', norm='rms', eps=1e-6):
        super().__init__()
        lead = (n_experts,) if n_experts else ()
        self.n_experts, self.activation, self.norm, self.eps = n_experts, activation, norm, eps
        self.w1, self.b1 = _weight(*lead, hidden, channels), torch.nn.Parameter(torch.zeros(*lead, hidden))
        self.w2, self.b2 = _weight(*lead, channels, hidden), torch.nn.Parameter(torch.zeros(*lead, channels))
        self.wg, self.bg = _weight(1, channels), torch.nn.Parameter(torch.zeros(1))
        self.scale = torch.nn.Parameter(torch.full((channels,), 0.5))
        self.post_weight = torch.nn.Parameter(torch.ones(channels))
        self.pre_weight = torch.nn.Parameter(torch.ones(channels))

    def forward(self, x, n, experts=None, weights=None):
        to = lambda p: p.to(x.dtype)  # noqa: E731
        if self.n_experts:
            order = expert_order(experts, self.n_experts)
            y = expert_dense(dispatch(n, order), to(self.w1), order.offsets, to(self.b1), self.activation)
            y = combine(expert_dense(y, to(self.w2), order.offsets, to(self.b2)), weights, order)
        else:
            y = dense(dense(n, to(self.w1), to(self.b1), self.activation), to(self.w2), to(self.b2))
        gate = torch.sigmoid(dense(n, to(self.wg), to(self.bg)))
        return block_norm(x, y, gate, to(self.scale), to(self.post_weight), to(self.pre_weight), self.eps, self.norm)


class NodeHead(torch.nn.Module):
    """Node features [N, features] to one value per node [N]: a linear embedding to ``channels``, its norm, ``layers``
    ``NodeFeedForward`` blocks and a linear readout of the last norm.  With ``n_experts`` a node's experts are given to
    ``forward`` (its element's index, [N] or [N, k]), or, with ``top_k``, chosen by a learned router per block: the top_k of a
    softmax over its projection of n, weighted by their probabilities."""

    def __init__(self, features, channels, hidden=None, layers=2, n_experts=0, top_k=0, activation='silu', norm='rms',
                 dtype=torch.float32):
        super().__init__()
        if top_k and not 1 <= top_k <= n_experts:
            raise ValueError(f'top_k must be between 1 and n_experts ({n_experts}), got {top_k}')
        self.top_k, self.dtype, self.n_experts = top_k, dtype, n_experts
        self.embed = _weight(channels, features)
        self.pre_weight = torch.nn.Parameter(torch.ones(channels))
        self.norm = norm
        self.blocks = torch.nn.ModuleList(NodeFeedForward(channels, hidden or 4 * channels, n_experts, activation, norm)
                                          for _ in range(layers))
        self.routers = torch.nn.ParameterList(_weight(n_experts, channels) for _ in range(layers if top_k else 0))
        self.readout = _weight(1, channels)

    def forward(self, feats, experts=None):
        if self.n_experts and not self.top_k:
            if experts is None:
                raise ValueError('a head with experts and no router needs the nodes\' experts')
            experts = experts if experts.dim() == 2 else experts[:, None]
        h = dense(feats.to(self.dtype), self.embed.to(self.dtype))
        h, n = block_norm(h, pre_weight=self.pre_weight.to(self.dtype), kind=self.norm)
        weights = None
        for i, block in enumerate(self.blocks):
            if self.top_k:
                p = torch.softmax(dense(n, self.routers[i].to(self.dtype)).float(), dim=1)
                weights, experts = torch.topk(p, self.top_k, dim=1)
            h, n = block(h, n, experts, weights)
        return dense(n, self.readout.to(self.dtype))[:, 0].float()


@torch.no_grad()
def node_features(model, batch, layer=-1):
    """The node features [N, D] that product block ``layer`` of a (patched) MACE model gives for a batch, detached: what a
    head is trained on.  The invariant channels come first."""
    kept = []
    hook = model.products[layer].register_forward_hook(lambda mod, args, out: kept.append(out))
    try:
        model(batch, compute_force=False)
    finally:
        hook.remove()
    return kept[0].detach().clone()
