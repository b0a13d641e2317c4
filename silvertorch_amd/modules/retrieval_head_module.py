"""Answers of a retrieval model from a score table held in 4 bits (no
reference counterpart)."""

from __future__ import annotations

import torch
import torch.nn as nn

import silvertorch_amd.ops._load_ops  # noqa: F401  (registers torch.ops.st)


class RetrievalHeadModule(nn.Module):
    """Holds a table of document embeddings in 4 bits as buffers (they follow
    ``.to(device)`` and ``state_dict``; a saved table loads into a new module),
    scores query vectors against it and gives the scores' log-probabilities
    among the documents that a filter lets pass.  The table's scores have no
    gradient: a backward pass through them is an error.

    Args:
        group_size: columns that share a scale (a multiple of 32).
        topk: alternatives returned per query (0 to 128).
        temperature: the scores are divided by it.
    """

    TABLE = ("packed", "scales", "zeros")

    def __init__(self, group_size: int = 32, topk: int = 10, temperature: float = 1.0) -> None:
        super().__init__()
        self.group_size = group_size
        self.topk = topk
        self.temperature = temperature
        self.register_buffer("packed", torch.empty((0, 0), dtype=torch.uint8))
        self.register_buffer("scales", torch.empty((0, 0), dtype=torch.float32))
        self.register_buffer("zeros", torch.empty((0, 0), dtype=torch.uint8))

    def set_table(self, packed: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor) -> None:
        self.packed, self.scales, self.zeros = packed, scales, zeros

    def set_embeddings(self, embeddings: torch.Tensor, symmetric: bool = True) -> None:
        """Packs document embeddings [num_docs, dim] into the table."""
        self.set_table(*torch.ops.st.int4_quantize(embeddings.detach(), self.group_size, symmetric))

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
