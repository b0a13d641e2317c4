"""A query tower: residual feed-forward layers with layer norm and dropout, as
it is trained, and the same tower with its weights in 8 bits, as it is served
(no reference counterpart)."""

from __future__ import annotations

import torch
import torch.nn as nn

import silvertorch_amd.ops._load_ops  # noqa: F401  (registers torch.ops.st)


class QueryTowerModule(nn.Module):
    """Maps query features [..., features] to embeddings [..., dim].

    ``h = in(dropout(x))``, then per layer ``h = h + dropout(down(relu(up(norm(h)))))``, then ``out(norm(h))``.
    A layer's end and the next norm are one pass (``dropout_add_layer_norm``).  Dropout stores no mask: it draws from
    ``rng`` (seed, next offset), a buffer on the module's device that every training pass advances, also when a graph
    replays it.  A pass that is computed twice (activation checkpointing) is given its state, for both to drop the same
    elements: ``checkpoint(tower, x, tower.next_state(), use_reentrant=False)``.  Without one it is refused where it is
    computed again, in the backward pass.

    Args:
        features: columns of the input.
        dim: columns of the embeddings.
        width: columns of the residual stream, 1 to 32768.
        layers: feed-forward layers, each ``expand`` times as wide inside.
        dropout: share of a layer's results (and of the input's features) that training drops.
        seed: of dropout's numbers; ranks of a data-parallel job take one each (and keep this buffer their own).
    """

    def __init__(self, features: int, dim: int, width: int, layers: int = 2, expand: int = 4, dropout: float = 0.1,
                 eps: float = 1e-5, seed: int = 0) -> None:
        super().__init__()
        self.dropout = dropout
        self.eps = eps
        self.enter = nn.Linear(features, width)
        self.up = nn.ModuleList(nn.Linear(width, expand * width) for _ in range(layers))
        self.down = nn.ModuleList(nn.Linear(expand * width, width) for _ in range(layers))
        self.norm_weights = nn.ParameterList(nn.Parameter(torch.ones(width)) for _ in range(layers + 1))
        self.norm_biases = nn.ParameterList(nn.Parameter(torch.zeros(width)) for _ in range(layers + 1))
        self.leave = nn.Linear(width, dim)
        self.register_buffer("rng", torch.tensor([seed, 0], dtype=torch.int64))
        # one state a pass for each place that drops
        self.register_buffer("places", torch.stack([torch.zeros(layers + 1, dtype=torch.int64),
                                                    torch.arange(layers + 1)], 1), persistent=False)

    def next_state(self) -> torch.Tensor:
        """The state (int64 [2]) of one training pass; ``rng`` goes on to the next one's."""
        state = self.rng.clone()
        self.rng[1] += len(self.places)
        return state

    def forward(self, x: torch.Tensor, state: torch.Tensor | None = None) -> torch.Tensor:
        """`state`: dropout's of this pass, from `next_state`; without it, a training pass takes the next one."""
        ops = torch.ops.st
        p, states = 0.0, [None] * len(self.places)
        if self.training and self.dropout > 0:
            if state is None:
                if torch._C._current_graph_task_id() != -1:
                    raise RuntimeError("a training pass inside a backward pass (activation checkpointing computes it "
                                       "again) would drop other elements than its first run: give it a state, "
                                       "checkpoint(tower, x, tower.next_state())")
                state = self.next_state()
            elif state.shape != (2,):
                raise RuntimeError(f"state must hold seed and offset, got a tensor of {list(state.shape)}")
            p, states = self.dropout, (state + self.places).unbind()
            x = ops.dropout(x, p, states[0])
        h = self.enter(x)
        y = ops.layer_norm(h, self.norm_weights[0], self.norm_biases[0], self.eps)
        for i, (up, down) in enumerate(zip(self.up, self.down), 1):
            z = down(torch.relu(up(y)))
            y, h = ops.dropout_add_layer_norm(z, h, self.norm_weights[i], self.norm_biases[i], p, states[i], self.eps)
        return self.leave(y)


class Int8Linear(nn.Module):
    """A linear layer whose weight is held in 8 bits, a scale for each output.  The input is taken to 8 bits on the way, a
    scale for each row, or comes as codes and scales.  It has no gradient.  Scales and bias stay float32 whatever the
    module is converted to."""

    def __init__(self, linear: nn.Linear) -> None:
        super().__init__()
        codes, scales = torch.ops.st.int8_quantize(linear.weight.detach())
        self.register_buffer("codes", codes)
        self.register_buffer("scales", scales)
        self.register_buffer("bias", None if linear.bias is None else linear.bias.detach().float())

    def _apply(self, fn, recurse=True):
        held = self.scales, self.bias
        super()._apply(fn, recurse)
        if self.scales.dtype != torch.float32:
            self.scales, self.bias = (t if t is None else t.to(self.scales.device) for t in held)
        return self

    def forward(self, x: torch.Tensor, x_scales: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
        return torch.ops.st.int8_matmul(self.codes, self.scales, x, x_scales, self.bias, out_dtype)


class PackedQueryTowerModule(nn.Module):
    """A trained :class:`QueryTowerModule` for serving: weights in 8 bits, each norm's result straight in 8 bits."""

    def __init__(self, tower: QueryTowerModule) -> None:
        super().__init__()
        self.eps = tower.eps
        self.enter = Int8Linear(tower.enter)
        self.up = nn.ModuleList(Int8Linear(m) for m in tower.up)
        self.down = nn.ModuleList(Int8Linear(m) for m in tower.down)
        self.leave = Int8Linear(tower.leave)
        for i, (w, b) in enumerate(zip(tower.norm_weights, tower.norm_biases)):
            self.register_buffer(f"norm_weight{i}", w.detach().clone())
            self.register_buffer(f"norm_bias{i}", b.detach().clone())

    def _norm(self, h: torch.Tensor, i: int):
        return torch.ops.st.layer_norm_int8(h, getattr(self, f"norm_weight{i}"), getattr(self, f"norm_bias{i}"), self.eps)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        h = self.enter(x)
        y, scales = self._norm(h, 0)
        for i, (up, down) in enumerate(zip(self.up, self.down), 1):
            h = h + down(torch.relu(up(y, scales, h.dtype)))
            y, scales = self._norm(h, i)
        return self.leave(y, scales, h.dtype)
