"""One block of a Gated DeltaNet model, with the parameter names and the call signature of the reference's ``GatedDeltaNetBlock``
(fla/models/gated_deltanet/modeling_gated_deltanet.py): normalisation, token mixing, normalisation of the residual stream that the mixing is added to, gated
feed-forward block.  Normalisations, the addition in front of the second one and the feed-forward block run in this package's HIP kernels, forward and backward; the
last addition is torch's; the mixing layer is ``GatedDeltaNet`` with its caches and its modes."""
from __future__ import annotations

import contextlib

import torch
import torch.nn as nn

from fla_hip.layers.gated_deltanet import GatedDeltaNet
from fla_hip.modules import GatedMLP, RMSNorm


class GatedDeltaNetBlock(nn.Module):

    def __init__(
        self,
        hidden_size: int = 2048,
        hidden_ratio: int | None = 4,
        intermediate_size: int | None = None,
        hidden_act: str = 'swish',
        norm_eps: float = 1e-6,
        layer_idx: int | None = None,
        **layer_kwargs,
    ):
        """``layer_kwargs``: what ``GatedDeltaNet`` takes besides its hidden size, its index and its norm's eps."""
        super().__init__()
        self.layer_idx = layer_idx
        self.attn_norm = RMSNorm(hidden_size, eps=norm_eps)
        self.attn = GatedDeltaNet(hidden_size=hidden_size, layer_idx=layer_idx, norm_eps=norm_eps, **layer_kwargs)
        self.mlp_norm = RMSNorm(hidden_size, eps=norm_eps)
        self.mlp = GatedMLP(hidden_size, hidden_ratio=hidden_ratio, intermediate_size=intermediate_size, hidden_act=hidden_act)

    def forward(
        self,
        hidden_states: torch.Tensor,
        attention_mask: torch.Tensor | None = None,
        past_key_values=None,
        use_cache: bool | None = False,
        output_attentions: bool | None = False,
        **kwargs,
    ):
        # (as in the layer: outside of training no graph is built)
        with contextlib.nullcontext() if self.training else torch.no_grad():
            residual = hidden_states
            hidden_states, attentions, past_key_values = self.attn(
                hidden_states=self.attn_norm(hidden_states), attention_mask=attention_mask, past_key_values=past_key_values, use_cache=use_cache,
                output_attentions=output_attentions, **kwargs)
            hidden_states, residual = self.mlp_norm(hidden_states, residual, True)
            return residual + self.mlp(hidden_states), attentions, past_key_values
