"""IdentityMapper: passes its kwargs through (reference feature_extractors/identity_mapper.py:6-11)."""
import torch

from ... import ops
from .builder import FEATURE_EXTRACTORS


@FEATURE_EXTRACTORS.register_module()
class IdentityMapper(torch.nn.Module):
    """dropout (0: the reference's mapper): probability of dropping an entry of the `global_codes` that it passes on, in
    training mode (module.train()), for codes that the caller computes; CodeTable does it for those that it learns. A step
    that is captured into a graph then passes `rng_base` (ops.dropout) beside the codes."""

    def __init__(self, dropout: float = 0.0):
        super().__init__()
        if not 0.0 <= dropout <= 1.0:
            raise ValueError(f"IdentityMapper: dropout probability {dropout} is not in [0, 1]")
        self.dropout = dropout

    def forward(self, **kwargs):
        if self.dropout > 0.0:
            base = kwargs.pop("rng_base", None)
            if self.training and kwargs.get("global_codes") is not None:
                kwargs["global_codes"] = ops.dropout(kwargs["global_codes"], self.dropout, rng_base=base)
        return kwargs
