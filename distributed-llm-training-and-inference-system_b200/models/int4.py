"""Projections of the GPT family whose weights stay in 4 bits for serving, as the ``int4`` quantiser (io/quantize.py) writes them: a quarter of the bytes that a decoding
step reads (``ops.functional.linear_int4``).  What the quantiser leaves in the source precision (embeddings, norms, widths that are no multiple of its groups) stays
as it is.

Reference: quantisation is an option of a stub command (llmctl/cli/commands/export.py:17)."""
from __future__ import annotations

from typing import Dict, Optional

import torch
import torch.nn as nn

from ..io.quantize import INT4_GROUP, SCALE_SUFFIX, Int4GroupQuantizer
from ..ops import functional as ops
from ..parallel import tp as tpl


class Int4Linear(nn.Module):
    """``x @ W.T`` for codes [N, K / 2] and scales [N, K / 128]."""

    def __init__(self, weight: torch.Tensor, scale: torch.Tensor):
        super().__init__()
        self.register_buffer("weight", weight)
        self.register_buffer("scale", scale)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return ops.linear_int4(x, self.weight, self.scale)

    def swiglu(self, x: torch.Tensor) -> torch.Tensor:
        """The gated MLP's first half, for packed gate | up rows."""
        return ops.linear_swiglu_int4(x, self.weight, self.scale)


def _fit(codes: torch.Tensor, scale: torch.Tensor, rows: int, width: int) -> bool:
    return (codes.dtype == torch.uint8 and codes.shape == (rows, width // 2) and scale.dtype == torch.float16 and width % INT4_GROUP == 0
            and scale.shape == (rows, width // INT4_GROUP))


def hold_in_int4(model: nn.Module, codes: Optional[Dict[str, torch.Tensor]] = None) -> int:
    """Puts an ``Int4Linear`` in the place of every projection of ``model`` that the quantiser takes (a head of its own among them); returns how many.  ``codes``:
    tensors of an ``int4`` artifact by name, used as they are; a projection that is not among them, or not as its codes and scales would be, is quantised from its weights."""
    codes, quantiser, done = codes or {}, Int4GroupQuantizer(), 0
    for path in [p for p, m in model.named_modules() if isinstance(m, (tpl.ColumnParallelLinear, tpl.RowParallelLinear))]:
        module = model.get_submodule(path)          # (one at a time: what is replaced gives its weights back)
        name, device = path + ".weight", module.weight.device
        got = {k: codes[k] for k in (name, name + SCALE_SUFFIX) if k in codes}
        if len(got) != 2 or not _fit(*got.values(), *module.weight.shape):
            got = quantiser.quantize({name: module.weight.detach()})
        if name + SCALE_SUFFIX not in got:
            continue
        parent = model.get_submodule(path.rpartition(".")[0])
        setattr(parent, path.rpartition(".")[2], Int4Linear(got[name].to(device), got[name + SCALE_SUFFIX].to(device)))
        done += 1
    return done
