"""CodeTable: learned global codes for the conditional NeRFMLP (latent_dim > 0), looked up by id.

The reference's conditional MLP takes `global_codes` from its caller (nerf_mlp.py:158-163; tests/test_pipeline.py:37-64
passes them through an IdentityMapper). This extractor holds the codes as a parameter instead, one row an image (or frame,
lighting, speaker ...), and trains them with the MLPs: the pipeline passes it the ids, it returns the codes."""
from __future__ import annotations

from typing import Optional

import torch

from ... import ops
from .builder import FEATURE_EXTRACTORS


@FEATURE_EXTRACTORS.register_module()
class CodeTable(torch.nn.Module):
    """{global_codes: dropout(scale * table[ids])} of the ids [B] passed to the pipeline under `ids_key`.

    num_codes, latent_dim: the table. scale: multiplies the codes (and their gradient). dropout: probability of dropping
    an entry of a code in training mode (module.train()); evaluation looks the codes up as they are. padding_idx: a row
    that stays as it is (it starts at zero). Rows start as N(0, init_std). A step that is captured into a graph with dropout
    passes `rng_base` (ops.dropout) beside the ids."""

    def __init__(self, num_codes: int, latent_dim: int, scale: float = 1.0, dropout: float = 0.0,
                 padding_idx: Optional[int] = None, init_std: float = 0.01, ids_key: str = "image_ids"):
        super().__init__()
        if num_codes < 1 or latent_dim < 1:
            raise ValueError("CodeTable needs num_codes >= 1 and latent_dim >= 1")
        if not 0.0 <= dropout <= 1.0:
            raise ValueError(f"CodeTable: dropout probability {dropout} is not in [0, 1]")
        if padding_idx is not None and not -num_codes <= padding_idx < num_codes:
            raise ValueError(f"CodeTable: padding_idx {padding_idx} is outside {num_codes} codes")
        self.num_codes, self.latent_dim = num_codes, latent_dim
        self.scale, self.dropout, self.padding_idx, self.ids_key = scale, dropout, padding_idx, ids_key
        self.table = torch.nn.Parameter(torch.randn(num_codes, latent_dim) * init_std)
        if padding_idx is not None:
            self.table.data[padding_idx] = 0.0

    def forward(self, **kwargs):
        ids = kwargs.get(self.ids_key)
        if ids is None:
            raise KeyError(f"CodeTable needs `{self.ids_key}`")
        ids = torch.as_tensor(ids)
        if ids.dtype.is_floating_point or ids.dtype.is_complex or ids.dtype == torch.bool:
            raise TypeError(f"CodeTable: `{self.ids_key}` must be integers, got {ids.dtype}")
        if ids.dim() != 1:
            raise ValueError(f"CodeTable: `{self.ids_key}` must be [B], got {tuple(ids.shape)}")
        on_host = ids.device.type == "cpu"
        if on_host and ids.numel() and not (0 <= int(ids.min()) and int(ids.max()) < self.num_codes):
            raise IndexError(f"CodeTable: an id lies outside {self.num_codes} codes")
        ids = ids.to(self.table.device, torch.int64)
        codes = ops.embedding(self.table, ids, scale=self.scale, padding_idx=self.padding_idx,
                              dropout=self.dropout if self.training else 0.0, rng_base=kwargs.get("rng_base"),
                              check=not on_host)
        return {"global_codes": codes}
