"""Qwen3-style decoder whose feed-forward layers are top-k routed mixtures of SwiGLU experts.

Not in the reference (its registry holds the dense model only; expert parallelism is an empty file there).  It exists
so that the expert-parallel layer (``parallel/expert_parallel.py``) has a model the config can select: every block
keeps the dense model's attention and norms and swaps the MLP for ``MoELayer``.  The blocks run the PyTorch path
(``impl`` is fixed to "torch"); ``experts: "grouped"`` runs the feed-forwards on the sm_100a operators of ``ops/moe.py``
instead of batched library products over padded buffers, and ``act_bits: 8`` keeps their gate and up in 8 bits between the
passes.  ``router`` ({"score", "groups", "top_groups", "group_scores", "normalize", "scale", "bias_rate"}) chooses experts by scores, with a bias that
the Trainer moves after every step; ``embedding: "sorted"`` looks tokens up with ``ops/embedding.py``, whose gradient sums a
token's rows in a fixed order, and ``embed_scale`` multiplies the rows.

With ``mesh: {"dp": D, "ep": E}`` the Trainer calls ``shard_experts``: rank r of an ``ep`` group keeps experts
[r E_total / E, (r + 1) E_total / E) of every layer, tokens travel to their experts' owners and back through the
even-split all-to-all, and every rank of the group reads different rows (the axis is also a data axis).
"""

from __future__ import annotations

import torch
import torch.nn as nn

from torchure_b200.core.collective import all_reduce
from torchure_b200.models.qwen3 import Qwen3, RMSNorm
from torchure_b200.ops.embedding import embedding
from torchure_b200.parallel.expert_parallel import MoELayer


class TokenEmbedding(nn.Embedding):
    """The token table `like`, the same parameter, with rows times `scale`; `by_sorting`: looked up by ``ops/embedding.py``.  A module, so that
    wrappers that hook its forward pass (sharded parameters, pipeline stages) find it where a plain table would be."""

    def __init__(self, like: nn.Embedding, scale: float, by_sorting: bool):
        super().__init__(*like.weight.shape, _weight=like.weight.detach())
        self.weight = like.weight
        self.scale, self.by_sorting = float(scale), by_sorting

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        if self.by_sorting:
            return embedding(ids, self.weight, self.scale)
        h = super().forward(ids)
        return h if self.scale == 1.0 else h * self.scale


class Qwen3MoE(Qwen3):
    def __init__(self, num_layers: int, num_heads: int, num_kv_heads: int, emb_dim: int, head_dim: int | None,
                 vocab_size: int, num_experts: int, top_k: int = 2, moe_ffn_dim: int | None = None,
                 capacity_factor: float = 2.0, aux_loss_coef: float = 0.01, ffn_dim: int | None = None,
                 norm_eps: float = 1e-6,
                 rope_theta: float = 1_000_000.0, qk_norm: bool = True, tie_embeddings: bool = True,
                 impl: str = "torch", experts: str = "capacity", act_bits: int = 16, router: dict | None = None,
                 embedding: str = "torch", embed_scale: float = 1.0):
        super().__init__(num_layers=num_layers, num_heads=num_heads, num_kv_heads=num_kv_heads, emb_dim=emb_dim,
                         head_dim=head_dim, vocab_size=vocab_size, ffn_dim=ffn_dim, norm_eps=norm_eps,
                         rope_theta=rope_theta, qk_norm=qk_norm, tie_embeddings=tie_embeddings, impl="torch")
        if embedding not in ("torch", "sorted"):
            raise ValueError(f'Qwen3MoE: the embedding is "torch" or "sorted", not {embedding!r}')
        width = moe_ffn_dim if moe_ffn_dim is not None else self.cfg["ffn_dim"]
        self.cfg.update(num_experts=num_experts, top_k=top_k, moe_ffn_dim=width, capacity_factor=capacity_factor,
                        aux_loss_coef=aux_loss_coef, experts=experts, act_bits=act_bits, router=router,
                        embedding=embedding, embed_scale=embed_scale)
        self.token_emb = TokenEmbedding(self.token_emb, embed_scale, embedding == "sorted")
        self.aux_loss_coef = aux_loss_coef
        for block in self.blocks:
            block.ffn = MoELayer(emb_dim, width, num_experts, top_k, capacity_factor, experts=experts, act_bits=act_bits,
                                 router=router)

    @torch.no_grad()
    def init_weights(self, std: float = 0.02) -> None:
        """The dense model's scheme; the stacked expert matrices count as matrices, and every expert's down
        projection gets the residual-stream scaling (2L)^-1/2."""
        for m in self.modules():
            if isinstance(m, (nn.Linear, nn.Embedding)):
                nn.init.normal_(m.weight, mean=0.0, std=std)
            elif isinstance(m, MoELayer):
                for w in (m.w_gate, m.w_up, m.w_down):
                    nn.init.normal_(w, mean=0.0, std=std)
            elif isinstance(m, RMSNorm):
                nn.init.ones_(m.weight)
        scale = (2 * len(self.blocks)) ** -0.5
        for b in self.blocks:
            b.gqa.o_proj.weight.mul_(scale)
            b.ffn.w_down.mul_(scale)

    @torch.no_grad()
    def balance_routers(self, mesh=None, dim: str | None = None) -> None:
        """After a training step: every router's bias against the choices counted since the last call, over all ranks of `dim`."""
        layers = [b.ffn for b in self.blocks if b.ffn.bias_rate]
        if not layers:
            return
        counts = torch.stack([layer.router_counts for layer in layers])
        if mesh is not None and mesh.size(dim) > 1:
            wide = counts.long()
            all_reduce(wide, mesh, dim, "sum")
            counts = wide.clamp_max(2 ** 31 - 1).int()
        for layer, mine in zip(layers, counts):
            layer.balance(mine)

    def aux_loss(self) -> torch.Tensor:
        """Mean over the layers of the routers' load-balancing terms of the LAST forward pass; the objective adds
        ``aux_loss_coef`` times this to the language-model loss."""
        terms = [b.ffn.aux_loss for b in self.blocks]
        return torch.stack(terms).mean()

    def fused_param_groups(self):
        return [(b.gqa.q_proj.weight, b.gqa.k_proj.weight, b.gqa.v_proj.weight) for b in self.blocks]

    def shard_experts(self, mesh, dim: str = "ep") -> None:
        for b in self.blocks:
            b.ffn.shard_(mesh, dim)

    def expert_params(self) -> list[nn.Parameter]:
        return [w for b in self.blocks for w in (b.ffn.w_gate, b.ffn.w_up, b.ffn.w_down)]
