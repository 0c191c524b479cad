"""Parameter-holding layers with the reference's names and init (net_layers.py:3-49), and the gated
linear recurrence layer.

ConvNorm / LinearNorm keep `.conv` / `.linear_layer` (torch Conv1d / Linear) so state_dict keys,
shapes and Xavier-uniform init match the reference exactly; their arithmetic never runs through
torch: the Generator calls the HIP kernels in autovc_amd.ops on these parameters.
"""
import math

import torch
import torch.nn as nn

from .. import ops


class LinearNorm(nn.Module):
    """Linear layer holder, xavier_uniform init with `w_init_gain` (net_layers.py:3-20)."""

    def __init__(self, in_dim, out_dim, bias=True, w_init_gain="linear"):
        super().__init__()
        self.linear_layer = nn.Linear(in_dim, out_dim, bias=bias)
        nn.init.xavier_uniform_(self.linear_layer.weight, gain=nn.init.calculate_gain(w_init_gain))


class ConvNorm(nn.Module):
    """Conv1d holder, xavier_uniform init with `w_init_gain` (net_layers.py:23-49)."""

    def __init__(self, in_channels, out_channels, kernel_size=1, stride=1, padding=None, dilation=1,
                 bias=True, w_init_gain="linear"):
        super().__init__()
        if padding is None:
            assert kernel_size % 2 == 1
            padding = int(dilation * (kernel_size - 1) / 2)
        if (kernel_size, stride, padding, dilation) != (5, 1, 2, 1):
            raise NotImplementedError("the HIP Conv1d implements the Generator's k=5, stride 1, pad 2")
        self.conv = nn.Conv1d(in_channels, out_channels, kernel_size=kernel_size, stride=stride,
                              padding=padding, dilation=dilation, bias=bias)
        nn.init.xavier_uniform_(self.conv.weight, gain=nn.init.calculate_gain(w_init_gain))


class LSTMParams(nn.Module):
    """Holds nn.LSTM's parameters under nn.LSTM's names (weight_ih_l{k}[_reverse], ...) and its
    default U(+-1/sqrt(H)) init, without nn.LSTM's cuDNN/MIOpen weight flattening."""

    def __init__(self, input_size, hidden_size, num_layers=1, batch_first=True, bidirectional=False):
        super().__init__()
        self.input_size, self.hidden_size, self.num_layers = input_size, hidden_size, num_layers
        self.batch_first, self.bidirectional = batch_first, bidirectional
        D = 2 if bidirectional else 1
        for l in range(num_layers):
            for sfx in ([""] + (["_reverse"] if bidirectional else [])):
                din = input_size if l == 0 else hidden_size * D
                self.register_parameter(f"weight_ih_l{l}{sfx}", nn.Parameter(torch.empty(4 * hidden_size, din)))
                self.register_parameter(f"weight_hh_l{l}{sfx}", nn.Parameter(torch.empty(4 * hidden_size, hidden_size)))
                self.register_parameter(f"bias_ih_l{l}{sfx}", nn.Parameter(torch.empty(4 * hidden_size)))
                self.register_parameter(f"bias_hh_l{l}{sfx}", nn.Parameter(torch.empty(4 * hidden_size)))
        self.reset_parameters()

    def reset_parameters(self):
        stdv = 1.0 / math.sqrt(self.hidden_size)
        for p in self.parameters():
            nn.init.uniform_(p, -stdv, stdv)

    def layer(self, l, reverse=False):
        sfx = "_reverse" if reverse else ""
        return (getattr(self, f"weight_ih_l{l}{sfx}"), getattr(self, f"weight_hh_l{l}{sfx}"),
                getattr(self, f"bias_ih_l{l}{sfx}"), getattr(self, f"bias_hh_l{l}{sfx}"))

    def flatten_parameters(self):  # encoder.py:74 calls this on nn.LSTM; nothing to do here
        return None


class GatedRecurrence(nn.Module):
    """A gated linear recurrence layer over time-major frames [T*B][C]: one projection to the gates
    (f, c, o of each direction, as rows [D][3][H] of `weight_ih`), then ops.gated_recurrence.  It
    stands where an nn.LSTM layer stands (decoder.py:37, encoder.py:51) when time is long: its cost
    does not grow with the number of steps in sequence.

    Initialised as LSTMParams (U(+-1/sqrt(H))), with the forget gates' bias raised by `forget_bias`
    so that a fresh layer remembers."""

    def __init__(self, input_size, hidden_size, bidirectional=False, reverse=False, forget_bias=1.0):
        super().__init__()
        if bidirectional and reverse:
            raise ValueError("a layer is bidirectional or reverse, not both")
        if input_size % 4 or hidden_size % 4:
            raise ValueError("the projection's products take widths that are multiples of 4")
        self.input_size, self.hidden_size = input_size, hidden_size
        self.dirs = 3 if bidirectional else 2 if reverse else 1
        D = 2 if bidirectional else 1
        self.weight_ih = nn.Parameter(torch.empty(D * 3 * hidden_size, input_size))
        self.bias_ih = nn.Parameter(torch.empty(D * 3 * hidden_size))
        stdv = 1.0 / math.sqrt(hidden_size)
        nn.init.uniform_(self.weight_ih, -stdv, stdv)
        nn.init.uniform_(self.bias_ih, -stdv, stdv)
        with torch.no_grad():
            self.bias_ih.view(D, 3, hidden_size)[:, 0].add_(forget_bias)

    def forward(self, x, T, B, h0=None, lengths=None):
        """x [T*B][input_size] -> (y [T*B][D*H], last states [D][B][H]); see ops.gated_recurrence."""
        return ops.gated_recurrence(self._gates(x), T, B, h0, lengths, self.dirs)

    @torch.no_grad()
    def step(self, x, state):
        """One frame of a forward layer, state [B][H] updated in place: x [B][input_size] -> y [B][H]."""
        if self.dirs != 1:
            raise ValueError("only a forward layer can be stepped")
        return ops.gated_recurrence_step(self._gates(x), state, out_state=state)[0]

    def _gates(self, x):
        if x.shape[0] == 0:  # no frame: nothing to launch, and no gradient but zero
            return nn.functional.linear(x, self.weight_ih, self.bias_ih)
        return ops.Linear.apply(x, self.weight_ih, self.bias_ih)
