"""``DistSAGEConvGrad`` (super_gnn/layers/sageconv.py:15-89): the caller of the hot
path.  Mean aggregation = Aggregator (sum) / in_degrees, then two bias-free
linear maps and a bias.  Plain ``torch.nn`` (the reference derives from a
torch_geometric fork only for the ``Linear`` / ``MessagePassing`` names)."""
from __future__ import annotations

import torch
from torch import Tensor
from torch.nn import Linear, Parameter

from ..aggregator import Aggregator
from ..time_recorder import TimeRecorder
from .functional import linear


class DistSAGEConvGrad(torch.nn.Module):
    def __init__(self, in_channels: int, out_channels: int, num_bits: int, is_pre_delay: bool,
                 add_self_loops: bool = False, normalize: bool = True, bias: bool = True, **kwargs):
        super().__init__()
        self.in_channels = in_channels
        self.out_channels = out_channels
        self.add_self_loops = add_self_loops
        self.normalize = normalize
        self.num_bits = num_bits
        self.is_pre_delay = is_pre_delay
        self.checkpoint_bits = 32  # 8: the inputs of the two linear maps are kept in 8 bits for the backward pass
        self.lin_neigh = Linear(in_channels, out_channels, bias=False)
        self.lin_self = Linear(in_channels, out_channels, bias=False)
        if bias:
            self.bias = Parameter(torch.zeros(out_channels))
        else:
            self.register_parameter("bias", None)

    def reset_parameters(self):
        gain = torch.nn.init.calculate_gain("relu")
        torch.nn.init.xavier_uniform_(self.lin_neigh.weight, gain=gain)
        torch.nn.init.xavier_uniform_(self.lin_self.weight, gain=gain)

    def propagate(self, graph, local_nodes_feat, layer):
        return Aggregator.apply(graph, local_nodes_feat, layer, self.num_bits, self.is_pre_delay, self.training)

    def forward(self, graph, local_nodes_feat, layer) -> Tensor:
        with TimeRecorder.ctx.time_block("total_aggregator(outer)", is_record=False):
            out = self.propagate(graph, local_nodes_feat, layer)
        with TimeRecorder.ctx.time_block("Normalization", is_record=False):
            if self.normalize and not getattr(graph, "fold_mean", False):
                out /= graph.in_degrees  # otherwise the Aggregator has already applied 1 / in_degree
        with TimeRecorder.ctx.time_block("nn_operation", is_record=False):
            if self.checkpoint_bits == 32 or not out.is_cuda:
                out = self.lin_neigh(out)
                out += self.lin_self(local_nodes_feat)
            else:
                out = linear(out, self.lin_neigh.weight, self.checkpoint_bits)
                # features without a gradient stay with the caller anyway
                bits = self.checkpoint_bits if local_nodes_feat.requires_grad else 32
                out += linear(local_nodes_feat, self.lin_self.weight, bits)
        with TimeRecorder.ctx.time_block("add_bias", is_record=False):
            if self.bias is not None:
                out += self.bias
        return out
