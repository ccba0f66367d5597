"""Learned relative position bias of a sparse attention's edges: the per-edge, per-head ``bias`` that
:func:`torchgt_b200.sparse_graph_attention` takes, looked up by the bucket of the distance between an edge's ends
(kernels: ``csrc/position_bias.cu``; node: ``csrc/binding_block.cpp``).

    offset_e = position[source] - position[destination],   bias[e] = table[bucket(offset_e)]

Buckets of one direction, ``n`` of them: distances below ``n // 2`` have a bucket each; the others' borders are even steps of
the logarithm from there to ``max_distance``, and the last bucket takes everything from its border on.  With ``bidirectional``
the table's second half is for sources behind their destination (offset > 0); without it those count as distance 0.  The
borders are whole numbers, ``d ** steps >= max_distance ** j * exact ** (steps - j)``, so no rounding of a logarithm decides
about a distance."""
from __future__ import annotations

import functools
import operator
from typing import Optional

import torch

from . import _cabi
from .linear import untraced

_MOST_BUCKETS, _MOST_HEADS = 512, 256
_IDS = (torch.int64, torch.int32)


def bucket_borders(num_buckets: int, max_distance: int, bidirectional: bool) -> tuple:
    """The smallest distance of every bucket of one direction but the first."""
    return _borders(operator.index(num_buckets), operator.index(max_distance), bool(bidirectional))


@functools.lru_cache(maxsize=64)
def _borders(num_buckets, max_distance, bidirectional):
    count = num_buckets // 2 if bidirectional else num_buckets
    if num_buckets > _MOST_BUCKETS or count < 2 or (bidirectional and num_buckets % 2):
        raise ValueError(f"num_buckets must be {'even and 4' if bidirectional else '2'} to {_MOST_BUCKETS}; got {num_buckets}")
    exact = count // 2
    if not exact < max_distance < 2 ** 31:
        raise ValueError(f"max_distance must be above {exact}, the distances with a bucket of their own, and below 2^31; "
                         f"got {max_distance}")
    steps = count - exact
    borders = list(range(1, exact + 1))
    for j in range(1, steps):
        bound = max_distance ** j * exact ** (steps - j)
        low, high = exact, max_distance
        while low < high:                    # the smallest whole number whose power reaches the bound
            middle = (low + high) // 2
            low, high = (low, middle) if middle ** steps >= bound else (middle + 1, high)
        borders.append(low)
    return tuple(borders)


def _as_operations(table, edge_index, positions, borders, bidirectional):
    """The same from operations that tracers, compilers and ``torch.func`` can record."""
    source, destination = edge_index.long().unbind(0)
    outside = None
    if positions is not None:
        nodes = positions.shape[0]
        outside = (source < 0) | (source >= nodes) | (destination < 0) | (destination >= nodes)
        positions = positions.long() if nodes > 0 else positions.new_zeros(1).long()
        last = positions.shape[0] - 1            # no index reaches past it: on a GPU torch's error ends the process's context
        source, destination = positions[source.clamp(0, last)], positions[destination.clamp(0, last)]
    behind = source > destination
    distance = torch.maximum(source, destination) - torch.minimum(source, destination)
    distance = torch.where(distance < 0, torch.iinfo(torch.int64).max, distance)         # 2^63 and more
    if not bidirectional:
        distance = distance.masked_fill(behind, 0)
    bucket = torch.bucketize(distance, torch.tensor(borders, device=table.device), right=True)
    if bidirectional:
        bucket = bucket + behind.long() * (len(borders) + 1)
    bias = torch.nn.functional.embedding(bucket, table)
    return bias if outside is None else torch.where(outside.unsqueeze(-1), float("nan"), bias)


def edge_position_bias(table: torch.Tensor, edge_index: torch.Tensor, positions: Optional[torch.Tensor] = None,
                       max_distance: int = 128, bidirectional: bool = True) -> torch.Tensor:
    """``bias`` [E, H] fp32 of the edges in ``edge_index`` ([2, E] int64 or int32: sources, destinations), in its order.

    ``table`` is [num_buckets, H] fp32 (up to 512 buckets and 256 heads); ``positions`` [N] int64 or int32 holds the nodes'
    positions (None: a node's position is its id).  An edge with an id outside the positions gets NaN and has no part in the
    gradient: nothing waits for the GPU to raise.  The table's gradient is summed in a fixed order (the same bits every
    time; where it is itself differentiated it is torch's ``index_add``, whose order may change).  Raises if the tensors are not on one CUDA device: there is no CPU path."""
    if not isinstance(edge_index, torch.Tensor):
        raise TypeError("edge_index must be the [2, E] tensor of the edges: a SparseGraph has them in another order")
    tensors = [table, edge_index] + ([positions] if positions is not None else [])
    if not all(t.is_cuda for t in tensors):
        raise RuntimeError("torchgt_b200.edge_position_bias needs CUDA tensors (no CPU fallback)")
    if any(t.device != table.device for t in tensors):
        raise ValueError("table, edge_index and positions must be on one device")
    if table.dtype != torch.float32 or edge_index.dtype not in _IDS or (positions is not None and positions.dtype not in _IDS):
        raise TypeError("table must be float32, edge_index and positions int64 or int32")
    if table.dim() != 2 or not 1 <= table.shape[1] <= _MOST_HEADS:
        raise ValueError(f"table must be [num_buckets, heads] with 1 to {_MOST_HEADS} heads; got {tuple(table.shape)}")
    if edge_index.dim() != 2 or edge_index.shape[0] != 2:
        raise ValueError("edge_index must be [2, E]")
    if positions is not None and positions.dim() != 1:
        raise ValueError("positions must be [N]")
    borders = bucket_borders(table.shape[0], max_distance, bidirectional)
    if untraced(*tensors):               # under autocast too: nothing here is of a type that it changes
        bias = _cabi.native().edge_position_bias(table, edge_index, positions, borders, bool(bidirectional))
        if bias is not None:
            return bias
    return _as_operations(table, edge_index, positions, borders, bidirectional)


class RelativePositionBias(torch.nn.Module):
    """``bias = module(edge_index, positions)`` for :func:`torchgt_b200.sparse_graph_attention`, with a learnt table
    ``weight`` [num_buckets, num_heads]."""

    def __init__(self, num_heads: int, num_buckets: int = 32, max_distance: int = 128, bidirectional: bool = True):
        super().__init__()
        bucket_borders(num_buckets, max_distance, bidirectional)            # refuses what it cannot make
        self.num_heads, self.num_buckets = num_heads, num_buckets
        self.max_distance, self.bidirectional = max_distance, bool(bidirectional)
        self.weight = torch.nn.Parameter(torch.empty(num_buckets, num_heads))
        torch.nn.init.normal_(self.weight, std=0.02)

    def forward(self, edge_index: torch.Tensor, positions: Optional[torch.Tensor] = None) -> torch.Tensor:
        return edge_position_bias(self.weight, edge_index, positions, self.max_distance, self.bidirectional)

    def extra_repr(self) -> str:
        return (f"{self.num_heads}, num_buckets={self.num_buckets}, max_distance={self.max_distance}, "
                f"bidirectional={self.bidirectional}")
