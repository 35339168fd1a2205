from fla_hip.ops.attn.paged import paged_append, paged_attn, paged_keep

__all__ = ['paged_append', 'paged_attn', 'paged_keep']
