from fla_hip.ops.drafts.verify import verify_drafts

__all__ = ['verify_drafts']
