"""Answers of a retrieval model from a score table held in 4 or 8 bits (no
reference counterpart)."""

from __future__ import annotations

import torch
import torch.nn as nn

import silvertorch_amd.ops._load_ops  # noqa: F401  (registers torch.ops.st)


class RetrievalHeadModule(nn.Module):
    """Holds a table of document embeddings in 4 or 8 bits as buffers (they follow
    ``.to(device)`` and ``state_dict``; a saved table loads into a new module),
    scores query vectors against it and gives the scores' log-probabilities
    among the documents that a filter lets pass.  The table's scores have no
    gradient: a backward pass through them is an error.

    Args:
        group_size: columns that share a scale in 4 bits (a multiple of 32).
        topk: alternatives returned per query (0 to 128).
        temperature: the scores are divided by it.
        bits: 4, or 8: a document has one scale then, and queries are taken to
            8 bits too.  A loaded or set table is used as what it is.
    """

    TABLE = ("packed", "scales", "zeros")

    def __init__(self, group_size: int = 32, topk: int = 10, temperature: float = 1.0, bits: int = 4) -> None:
        super().__init__()
        if bits not in (4, 8):
            raise RuntimeError(f"bits must be 4 or 8, got {bits}")
        self.bits = bits
        self.group_size = group_size
        self.topk = topk
        self.temperature = temperature
        self.register_buffer("packed", torch.empty((0, 0), dtype=torch.uint8))
        self.register_buffer("scales", torch.empty((0, 0), dtype=torch.float32))
        self.register_buffer("zeros", torch.empty((0, 0), dtype=torch.uint8))

    def set_table(self, packed: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None) -> None:
        """What `int4_quantize` returns, or `int8_quantize` (without zeros)."""
        if zeros is None:
            zeros = torch.empty((0, 0), dtype=torch.uint8, device=packed.device)
        self.packed, self.scales, self.zeros = packed, scales, zeros

    def set_embeddings(self, embeddings: torch.Tensor, symmetric: bool = True) -> None:
        """Packs document embeddings [num_docs, dim] into the table; `symmetric` is for 4 bits."""
        if self.bits == 8:
            self.set_table(*torch.ops.st.int8_quantize(embeddings.detach()))
            return
        self.set_table(*torch.ops.st.int4_quantize(embeddings.detach(), self.group_size, symmetric))

    def _apply(self, fn, recurse=True):
        held = self.scales
        super()._apply(fn, recurse)
        if self.packed.dtype == torch.int8 and self.scales.dtype != torch.float32:
            self.scales = held.to(self.scales.device)  # an 8-bit table's stay float32
        return self

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys,
                              unexpected_keys, error_msgs):
        # The buffers take the saved table's sizes and the scales its type; they
        # stay on the module's device.
        for name in self.TABLE:
            saved = state_dict.get(prefix + name)
            cur = getattr(self, name)
            if isinstance(saved, torch.Tensor) and (saved.shape != cur.shape or saved.dtype != cur.dtype):
                setattr(self, name, torch.empty(saved.shape, dtype=saved.dtype, device=cur.device))
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys,
                                      unexpected_keys, error_msgs)

    def scores(self, query_embeddings: torch.Tensor) -> torch.Tensor:
        """float32[Q, num_docs]: products of query vectors [Q, dim] with the table."""
        if self.packed.dtype == torch.int8:
            return torch.ops.st.int8_matmul(self.packed, self.scales, query_embeddings, None, None, torch.float32)
        return torch.ops.st.int4_matvec(self.packed, self.scales, query_embeddings, self.group_size, self.zeros,
                                        torch.float32)

    def forward(self, query_embeddings: torch.Tensor, targets: torch.Tensor | None = None,
                packed_mask: torch.Tensor | None = None):
        """(logprobs[Q], entropy[Q], lse[Q], top_ids[Q, topk], top_logprobs[Q, topk]) over the documents whose bit
        is set in `packed_mask`, the packed search output (all without one); `targets` int64[Q] are the documents
        whose log-probability is wanted (0 without them)."""
        if targets is None:
            targets = torch.full((query_embeddings.shape[0],), -1, dtype=torch.int64, device=query_embeddings.device)
        return torch.ops.st.target_logprobs(self.scores(query_embeddings), targets, self.topk, packed_mask,
                                            self.temperature)
