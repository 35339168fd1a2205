"""The callers of the gated delta rule path: the Gated DeltaNet token-mixing layer, and the block of a model around it."""
from fla_hip.layers.gated_deltanet import GatedDeltaNet, LayerCache
from fla_hip.layers.gated_deltanet_block import GatedDeltaNetBlock

__all__ = ['GatedDeltaNet', 'GatedDeltaNetBlock', 'LayerCache']
