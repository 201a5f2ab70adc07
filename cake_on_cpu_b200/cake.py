"""``cake_linear`` on CUDA tensors.

Mirrors the reference's PyTorch binding: the autograd function and module of
python/cake.py:18-49 and the three products of src/linear.cpp (forward
y = x W^T + b at :12-49; backward dX = dY W and dW = dY^T X at :52-102), each
product being one cake_sgemm call.  Tensors stay on the GPU: the library is
handed device pointers, transposed operands are read where they lie (the weight
of the forward product and dY of the weight gradient; the reference makes
contiguous transposed copies at src/linear.cpp:22 and :76-80) and the bias is
added in the product's epilogue instead of a second pass (:44-46).

Around the layer: ``cake_muon``, an optimiser that moves its weight by orthogonalised updates, and
``cake_linear_q4``, the layer with its weight held in 4 bits.
"""
import os

import torch
from torch import nn
from torch.nn import Parameter

from . import api


def linear_cpp():
    """The compiled extension `linear_cpp` (csrc/linear.cpp, the counterpart of the reference's
    src/linear.cpp built by python/setup.py); None when it has not been built
    (`python -m cake_on_cpu_b200.build --linear`)."""
    if not os.path.exists(os.path.join(os.path.dirname(os.path.abspath(__file__)), "linear_cpp.so")):
        return None
    api.lib()
    from . import linear_cpp as ext
    return ext



def _rows(t):
    """A 2-D view whose rows are contiguous (copies only if they are not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def linear_forward(input, weight, bias=None):
    """y = input @ weight.T (+ bias), as linear_forward in src/linear.cpp:12-49."""
    x = _rows(input.reshape(-1, input.shape[-1]))
    out = api.cake_sgemm_ex(x, _rows(weight), trans_b=True, bias=None if bias is None else bias.contiguous())
    return out.reshape(*input.shape[:-1], weight.shape[0])


def linear_backward(grad_output, input, weight, bias=None):
    """(grad_input, grad_weight, grad_bias), as linear_backward in src/linear.cpp:52-102."""
    dy = _rows(grad_output.reshape(-1, grad_output.shape[-1]))
    x = _rows(input.reshape(-1, input.shape[-1]))
    grad_input = api.cake_sgemm_ex(dy, _rows(weight)).reshape(input.shape)
    grad_weight = api.cake_sgemm_ex(dy, x, trans_a=True)
    grad_bias = dy.sum(0) if bias is not None else None
    return grad_input, grad_weight, grad_bias


class cake_linear_function(torch.autograd.Function):
    """The autograd function of python/cake.py:18-31.  With the compiled extension present the three
    products go through `linear_cpp.forward / backward` exactly as there; without it the ctypes
    routines above compute the same products through the same C-ABI entry point."""

    @staticmethod
    def forward(ctx, data, weight, bias=None):
        ext = linear_cpp()
        if ext is not None and data.dim() == 2:
            output = ext.forward(data, weight, bias)
        else:
            output = linear_forward(data, weight, bias)
        ctx.save_for_backward(data, weight, bias)
        return output

    @staticmethod
    def backward(ctx, grad_output):
        data, weight, bias = ctx.saved_tensors
        ext = linear_cpp()
        if ext is not None and data.dim() == 2:
            gi, gw, gb = ext.backward(grad_output.contiguous(), data, weight, bias)
            return gi, gw, (gb if bias is not None else None)
        return linear_backward(grad_output, data, weight, bias)


class cake_linear(nn.Module):
    """Drop-in for the reference's ``cake_linear`` module (python/cake.py:33-49)."""

    def __init__(self, input_features, output_features, bias=True):
        super().__init__()
        self.input_features = input_features
        self.output_features = output_features
        self.weight = Parameter(torch.empty(output_features, input_features))
        if bias:
            self.bias = Parameter(torch.empty(output_features))
        else:
            self.register_parameter("bias", None)
        self.weight.data.uniform_(-0.1, 0.1)
        if bias:
            self.bias.data.uniform_(-0.1, 0.1)

    def forward(self, data):
        return cake_linear_function.apply(data, self.weight, self.bias)


def _even_rows(t):
    """The tensor with contiguous rows that are evenly spaced over all its leading dimensions (copies only if they are not)."""
    if t.is_contiguous() or t.dim() == 0:
        return t
    if t.dim() <= 2:
        t = _rows(t)
        return t if t.dim() < 2 or t.shape[0] < 2 or t.stride(0) >= t.shape[1] else t.contiguous()
    if t.stride(-1) == 1:
        try:
            if t.view(-1, t.shape[-1]).stride(0) >= t.shape[-1]:
                return t
        except RuntimeError:
            pass
    return t.contiguous()


class cake_linear_q4_function(torch.autograd.Function):
    """y = x W^T + b with W a ``Q4Weights``, and its gradients for x and b; the 4-bit weight itself has none.  As ``cake_linear``,
    it takes any strides."""

    @staticmethod
    def forward(ctx, data, weights, bias=None):
        ctx.weights, ctx.has_bias = weights, bias is not None
        return api.cake_q4_linear(_even_rows(data), weights, None if bias is None else bias.contiguous())

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output):
        dy = grad_output if grad_output.is_contiguous() else grad_output.contiguous()
        gi = api.cake_q4_linear_dx(dy, ctx.weights) if ctx.needs_input_grad[0] else None
        gb = None
        if ctx.has_bias and ctx.needs_input_grad[2]:
            gb = dy.reshape(-1, dy.shape[-1]).sum(0, dtype=torch.float32).to(dy.dtype)
        return gi, None, gb


class cake_linear_q4(nn.Module):
    """``cake_linear`` with its weight in 4 bits: for serving, and for training what lies in front of it.  The packed weight is a
    buffer (it moves with the module and is part of its state), the bias a parameter of the type of the activations.

    The state also says what the packed bytes hold (their number does not: sizes are padded, and scales of either type take two
    bytes).  Loading the state of another geometry raises and leaves the layer as it is; so does one that does not say it, but
    with ``strict=False``, where only the number of bytes is compared."""

    def __init__(self, weights, bias=None):
        super().__init__()
        if not isinstance(weights, api.Q4Weights):
            raise TypeError("the weights must be a Q4Weights object")
        self.input_features, self.output_features = weights.in_features, weights.out_features
        self._geometry = (weights.out_features, weights.in_features, weights.group, weights.scale_type, weights.has_zeros)
        self.register_buffer("packed", weights.packed)
        self._weights = weights
        if bias is None:
            self.register_parameter("bias", None)
        else:
            self.bias = Parameter(bias.detach().clone())

    @classmethod
    def from_linear(cls, layer, group=128, symmetric=True, scale_dtype=None):
        """The 4-bit form of a layer with ``weight`` (out_features, in_features) and ``bias``."""
        return cls(api.Q4Weights.quantize(layer.weight.detach(), group, symmetric, scale_dtype), layer.bias)

    @property
    def weights(self):
        if self._weights.packed is not self.packed:  # moved, or loaded
            self._weights = api.Q4Weights.from_packed(self.packed, *self._geometry)
        return self._weights

    def get_extra_state(self):
        return torch.tensor(self._geometry, dtype=torch.int64)

    def set_extra_state(self, state):
        pass  # compared before anything is loaded

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        state = state_dict.get(prefix + "_extra_state")
        if state is not None:
            theirs = tuple(int(v) for v in state)
            if theirs != tuple(int(v) for v in self._geometry):
                error_msgs.append("%s: the state holds weights of (out_features, in_features, group, scale type, has zeros) %s, the layer's are %s"
                                  % (prefix or "cake_linear_q4", theirs, tuple(int(v) for v in self._geometry)))
                return
        elif strict:
            missing_keys.append(prefix + "_extra_state")
            return
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)

    def forward(self, data):
        return cake_linear_q4_function.apply(data, self.weights, self.bias)


class cake_muon(torch.optim.Optimizer):
    """Steps weight matrices along the orthogonalisation of their momentum (``cake_muon_step``).  Takes matrices in float32 or
    bfloat16 on the GPU; the momentum is kept in float32.  ``scale`` None: sqrt(max(1, rows / cols)) of each matrix."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, scale=None, steps=5, coeffs=api.NS_COEFFS, eps=1e-7):
        if lr < 0 or not 0 <= momentum <= 1 or weight_decay < 0:
            raise ValueError("lr and weight_decay are not negative, momentum lies between 0 and 1")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, scale=scale, steps=steps,
                                      coeffs=tuple(coeffs), eps=eps))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() != 2:
                    raise ValueError("cake_muon takes matrices; give other parameters to another optimiser")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("cake_muon takes dense gradients")
                state = self.state[p]
                if "momentum" not in state:
                    state["momentum"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                api.cake_muon_step(p, _rows(p.grad), state["momentum"], group["lr"], group["momentum"], group["nesterov"], group["weight_decay"],
                                   group["scale"], group["steps"], group["coeffs"], group["eps"])
                torch.autograd.graph.increment_version(p)  # written behind autograd's back
        return loss

    def load_state_dict(self, state_dict):
        """As every optimiser's, but the momentum stays in float32 (it would be rounded to the type of its parameter)."""
        super().load_state_dict(state_dict)
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(ids, params):
            saved = state_dict["state"].get(i, {})
            if "momentum" in saved:
                self.state[p]["momentum"] = saved["momentum"].to(device=p.device, dtype=torch.float32, copy=True).contiguous()
