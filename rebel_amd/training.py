"""Operators of the value net's training on the GPU: what lies between its matrix products (layer normalisation, with the GELU
behind it) and between the backward pass and the optimizer (the gradients' norm and clipping).

    layer_norm, LayerNorm     forward and backward as HIP kernels (rbl_layer_norm_* of the C ABI)
    grad_norm, clip_grad_norm_  one norm over many tensors, two launches to clip them (rbl_grad_*)
    train_step                one step of a trainer: Net2(native=True) forward, loss, backward, clipping, optimizer

Everything runs on torch's current stream and can be captured into a HIP graph; there is no CPU path.  A refused argument
raises ValueError, a failed launch RuntimeError.  Results repeat bit by bit: no sum depends on timing.

Capturing a backward pass: no graph that was made outside the capture may still hold a leaf of it (layer_norm refuses such a
leaf; delete the outputs of the warm-up first).  torch.cuda.make_graphed_callables keeps its own warm-up's graph and is refused for
that reason; torch.cuda.graph around a whole step works.
"""
import torch
from torch import nn

from rebel_amd import capi

capi.lib()  # librebel_hip.so first, with its message if it has not been built
from rebel_amd import _train  # noqa: E402

ACTIVATIONS = {None: capi.ACT_NONE, "gelu": capi.ACT_GELU}


def layer_norm(x, weight=None, bias=None, eps=1e-5, activation=None):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension of x; activation "gelu": x/2 (1 + erf(x / sqrt 2))
    of that, in the same pass.

    x: float32, float16 or bfloat16 on the GPU, any leading dimensions, up to 2^30 columns.  weight, bias: None, or
    [x.size(-1)] of x's type or float32.  The result has x's type; statistics, sums and the activation are computed in 32 bits (where a
    row's sum of values or of squared deviations passes 3e38, it overflows).
    Differentiable once, backward, in x, weight and bias.  Rows may lie at any one distance from each other; a layout that one row distance
    does not describe is copied first.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f"layer_norm: activation must be None or 'gelu', not {activation!r}")
    if torch.jit.is_tracing():
        raise ValueError("layer_norm: a trace would keep its result as a constant; trace the LayerNorm module")
    return _train.layer_norm(x, weight, bias, eps, ACTIVATIONS[activation])


class LayerNorm(nn.Module):
    """layer_norm as a module, with its parameters under the usual names (weight, bias: the state_dict of a net that is trained
    with it loads anywhere); `activation` as there.

    A scripted or traced copy holds torch's own operators, so that a saved TorchScript file needs nothing of this package.
    """

    def __init__(self, normalized_shape, eps=1e-5, elementwise_affine=True, bias=True, activation=None, device=None, dtype=None):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"LayerNorm: activation must be None or 'gelu', not {activation!r}")
        shape = tuple(normalized_shape) if isinstance(normalized_shape, (tuple, list, torch.Size)) else (normalized_shape,)
        if len(shape) != 1 or shape[0] < 1:
            raise ValueError(f"LayerNorm: normalized_shape must be the size of the last dimension, not {normalized_shape}")
        self.normalized_shape, self.eps, self.activation = [int(shape[0])], float(eps), activation
        if elementwise_affine:
            self.weight = nn.Parameter(torch.ones(shape, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
        if elementwise_affine and bias:
            self.bias = nn.Parameter(torch.zeros(shape, device=device, dtype=dtype))
        else:
            self.register_parameter("bias", None)

    def forward(self, x):
        if torch.jit.is_scripting() or torch.jit.is_tracing():
            y = nn.functional.layer_norm(x, self.normalized_shape, self.weight, self.bias, self.eps)
            return y if self.activation is None else nn.functional.gelu(y)
        else:
            return layer_norm(x, self.weight, self.bias, self.eps, self.activation)

    def extra_repr(self):
        return (f"{self.normalized_shape[0]}, eps={self.eps}, elementwise_affine={self.weight is not None}, "
                f"bias={self.bias is not None}, activation={self.activation}")


def grad_norm(tensors, norm_type=2.0):
    """The norm (order 1, 2 or inf) of all values of `tensors` taken as one vector: a float32 scalar on their device.

    Sums are held in 64 bits.  float32, float16 and bfloat16 tensors may be mixed; all must be on one GPU.  The norm has no gradient:
    tensors that require one are refused unless under no_grad.
    """
    return _train.grad_norm(_as_list(tensors), float(norm_type))


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Scales the gradients of `parameters` in place by min(1, max_norm / (norm + 1e-6)) and returns grad_norm of them before.

    Parameters without a gradient are passed over; no gradient at all gives tensor(0.).  A norm that is not finite scales all the
    same (the formula's zeros and NaN; one that is finite in 64 bits alone is returned as inf and scales by what it is), unless
    error_if_nonfinite, which waits for the norm on the host and raises RuntimeError with the gradients as they were.  Gradients that
    share memory are refused; one with gaps between its values is copied.  They may be blocks of one buffer (its columns, say) or every
    k-th of its rows; where they lie between each other in no such order, they are refused too.
    """
    return _train.clip_grad_norm(_as_list(parameters), float(max_norm), float(norm_type), error_if_nonfinite)


def _as_list(tensors):
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def value_loss(net, query, values):
    """The trainer's loss (/root/reference/cfvpy/selfplay.py:135-152): the square of the error up to 1, then linear, averaged."""
    error = (values - net(query)).abs()
    return torch.where(error > 1, error * 2 - 1, error * error).mean(-1).mean()


def train_step(net, optimizer, query, values, max_grad_norm=None, loss=value_loss):
    """One step on a batch as ValuePrioritizedReplay.sample returns it (/root/reference/cfvpy/selfplay.py:418-439): forward, loss,
    backward, clipping to max_grad_norm (None: none), optimizer step.  Returns (loss, norm of the gradients before clipping),
    both on the GPU; nothing waits for them."""
    optimizer.zero_grad()
    value = loss(net, query, values)
    value.backward()
    grads = [p for p in net.parameters() if p.grad is not None]
    if max_grad_norm is None:
        norm = grad_norm([p.grad for p in grads])
    else:
        norm = clip_grad_norm_(grads, max_grad_norm)
    optimizer.step()
    return value.detach(), norm
