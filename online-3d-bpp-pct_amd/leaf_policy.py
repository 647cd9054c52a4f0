"""A pointer policy over the observation's nodes, built on the package's own attention: what `collect` and
`RolloutSlots.evaluate` take logits from.  The roles are those of the reference's encoder and decoder (attention_model.py,
graph_encoder.py): every node attends to the nodes that are there, then every leaf does, and a leaf's score is its logit."""
import torch

from .policy_ops import cross_attention


class LeafPolicy(torch.nn.Module):
    """all_nodes [N, I + L + 1, 9] -> logits [N, L].  `width` / `heads` must be a multiple of 8, 128 at most; `dtype` (float32,
    bfloat16 or float16) is that of the weights and the attention, the logits are float32."""

    def __init__(self, internal_node_holder, leaf_node_holder, width=64, heads=1, dtype=torch.float32, device=None):
        super().__init__()
        if width % heads or (width // heads) % 8 or width // heads > 128:
            raise ValueError("LeafPolicy: width / heads must be a multiple of 8 up to 128, not %d / %d" % (width, heads))
        self.holders, self.heads = (internal_node_holder, leaf_node_holder), heads
        kw = dict(dtype=dtype, device=device)
        kinds = torch.cat([torch.full((n,), i) for i, n in enumerate((internal_node_holder, leaf_node_holder, 1))])
        self.register_buffer("kind", kinds.to(device), persistent=False)  # placed box, leaf, the item to place
        self.kinds = torch.nn.Parameter(torch.zeros(3, width, **kw))
        self.embed = torch.nn.Linear(9, width, **kw)
        self.node_qkv = torch.nn.Linear(width, 3 * width, **kw)
        self.leaf_q = torch.nn.Linear(width, width, **kw)
        self.leaf_kv = torch.nn.Linear(width, 2 * width, **kw)
        self.score = torch.nn.Linear(width, 1, **kw)

    def forward(self, all_nodes):
        (i, l), n, h = self.holders, all_nodes.shape[0], self.heads
        d = self.embed.out_features // h
        if all_nodes.dim() != 3 or all_nodes.shape[1:] != (i + l + 1, 9):
            raise ValueError("LeafPolicy: observations must be [N, %d, 9], not %s" % (i + l + 1, tuple(all_nodes.shape)))
        mask = all_nodes[:, :, 8]
        x = self.embed(all_nodes.to(self.embed.weight.dtype)) + self.kinds[self.kind]
        q, k, v = self.node_qkv(x).view(n, i + l + 1, 3, h, d).unbind(2)
        x = x + cross_attention(q, k, v, key_mask=mask).flatten(2)
        leaves = x[:, i:i + l]
        k, v = self.leaf_kv(x).view(n, i + l + 1, 2, h, d).unbind(2)
        seen = cross_attention(self.leaf_q(leaves).view(n, l, h, d), k, v, key_mask=mask)
        return self.score(torch.tanh(leaves + seen.flatten(2))).squeeze(2).float()
