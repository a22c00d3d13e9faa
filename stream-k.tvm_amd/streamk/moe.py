"""A feed-forward layer of experts on the grouped products.

A router's logits choose `chosen` of `experts` for each token (`route_experts`); the tokens' rows are laid out by expert
(`dispatch_rows`), go through the experts' two products with the activation between them (`streamk_grouped`), and come back as the sum
that the router's weights make (`combine_rows`).  No size depends on who chose whom: nothing waits for the device, and a call can be
recorded into a graph.

16-bit weights are parameters, and the layer trains: the products have gradients without fused activation, so a call that autograd
records applies it as an operation of its own.  int8 weights have a scale for each row, mxfp4 weights one for each 32 of it; the tokens are
quantised before they are laid out (a token's row and scales once, not once for each of its experts) and the hidden rows after the activation.
"""
import math
import warnings

import torch

from .experts import MAX_CHOSEN, MAX_EXPERTS, check_scores, combine_rows, dispatch_rows, route_experts, streamk_grouped
from .int8 import quantize_int8
from .mxfp4 import quantize_mxfp4

# weight_format -> how rows are quantised, values to a byte of weights, values to a scale (0: the row's), the scales' type, what K is a multiple of
_QUANTIZED = {"int8": (quantize_int8, torch.int8, 1, 0, torch.float32, 16), "mxfp4": (quantize_mxfp4, torch.uint8, 2, 32, torch.uint8, 32)}
_ACTIVATIONS = {"relu": torch.nn.functional.relu, "gelu_tanh": lambda x: torch.nn.functional.gelu(x, approximate="tanh"), "silu": torch.nn.functional.silu}


class StreamKMoE(torch.nn.Module):
    """experts of  W_down activation(W_up x)  with W_up [intermediate, hidden] and W_down [hidden, intermediate]; x [..., hidden] in
    `dtype` (float16 or bfloat16; weight_format 'float16' and 'bfloat16' say it themselves, 'int8' and 'mxfp4' take float16 by default).

    scores, groups, chosen_groups, renormalize, scale: as route_experts takes them.  balance: the layer has a buffer `router_bias` (float32
    [experts], zeros at first) that experts are chosen by beside their scores; who balances their load sets it.  A cast of the layer rounds
    it as it does any buffer, with a warning: in bfloat16 steps of a thousandth vanish from a half on.  The rule's own float32 sum, copied
    into the buffer after each step, loses none; `layer.router_bias = layer.router_bias.float()` makes the buffer float32 again."""

    def __init__(self, hidden, intermediate, experts, chosen, *, activation="silu", weight_format="bfloat16", dtype=None, device=None, scores="softmax",
                 balance=False, groups=1, chosen_groups=1, renormalize=True, scale=1.0):
        super().__init__()
        if activation not in _ACTIVATIONS:
            raise ValueError("activation must be 'relu', 'gelu_tanh' or 'silu'")
        if weight_format not in ("float16", "bfloat16", *_QUANTIZED):
            raise ValueError("weight_format must be 'float16', 'bfloat16', 'int8' or 'mxfp4'")
        own = {"float16": torch.float16, "bfloat16": torch.bfloat16}.get(weight_format, dtype or torch.float16)
        if own not in (torch.float16, torch.bfloat16) or (dtype is not None and dtype != own):
            raise ValueError(f"weight_format '{weight_format}' does not go with {dtype}")
        step = _QUANTIZED[weight_format][-1] if weight_format in _QUANTIZED else 8
        if hidden % step or intermediate % step:
            raise ValueError(f"hidden and intermediate must be multiples of {step} with {weight_format} weights")
        if not 1 <= experts <= MAX_EXPERTS or not 1 <= chosen <= min(experts, MAX_CHOSEN):
            raise ValueError(f"1 to {MAX_EXPERTS} experts, of which 1 to {MAX_CHOSEN} are chosen: got {experts} and {chosen}")
        check_scores(experts, chosen, scores, groups, chosen_groups, scale)
        self.hidden, self.intermediate, self.experts, self.chosen = hidden, intermediate, experts, chosen
        self.activation, self.weight_format, self.dtype = activation, weight_format, own
        self.routing = dict(scores=scores, groups=groups, chosen_groups=chosen_groups, renormalize=renormalize, scale=scale)
        self.register_buffer("router_bias", torch.zeros(experts, dtype=torch.float32, device=device) if balance else None)
        shapes = {"up": (experts, intermediate, hidden), "down": (experts, hidden, intermediate)}
        if weight_format in _QUANTIZED:
            _, kind, packed, block, scale_kind, _ = _QUANTIZED[weight_format]
            self.register_buffer("router", torch.zeros(experts, hidden, dtype=own, device=device))
            for name, shape in shapes.items():
                self.register_buffer(name, torch.zeros(*shape[:2], shape[2] // packed, dtype=kind, device=device))
                scales = (*shape[:2], shape[2] // block) if block else shape[:2]
                self.register_buffer(name + "_scale", torch.zeros(scales, dtype=scale_kind, device=device))
        else:
            self.router = torch.nn.Parameter(torch.randn(experts, hidden, dtype=own, device=device) / math.sqrt(hidden))
            for name, shape in shapes.items():
                self.register_parameter(name, torch.nn.Parameter(torch.randn(shape, dtype=own, device=device) / math.sqrt(shape[2])))

    @classmethod
    def quantized(cls, layer, weight_format="int8"):
        """The int8 or mxfp4 layer of a 16-bit one, on its device."""
        if weight_format not in _QUANTIZED or layer.weight_format in _QUANTIZED:
            raise ValueError(f"a layer of 16-bit weights becomes one of 'int8' or 'mxfp4': got '{layer.weight_format}' and '{weight_format}'")
        m = cls(layer.hidden, layer.intermediate, layer.experts, layer.chosen, activation=layer.activation, weight_format=weight_format, dtype=layer.dtype,
                device=layer.up.device, balance=layer.router_bias is not None, **layer.routing)
        m.router.copy_(layer.router.detach())
        if layer.router_bias is not None:
            m.router_bias.copy_(layer.router_bias)
        for name in ("up", "down"):
            q, scale = _QUANTIZED[weight_format][0](getattr(layer, name).detach())
            getattr(m, name).copy_(q)
            getattr(m, name + "_scale").copy_(scale)
        return m

    def _apply(self, fn, *args, **kwargs):
        before = self.router_bias
        super()._apply(fn, *args, **kwargs)
        if before is not None and self.router_bias.dtype != before.dtype and self.router_bias.dtype in (torch.float16, torch.bfloat16):
            warnings.warn(f"StreamKMoE: router_bias has been rounded to {self.router_bias.dtype}; small steps added to it there are lost", stacklevel=3)
        return self

    def route(self, x):
        """The route of x [T, hidden].  The router's product is one group of all rows.  Its logits come in x's type, as those of a linear
        layer in that type do: a half unit of a logit, 2^-8 of it in bfloat16, moves its token's weights by about as much and decides
        between experts that are that close.  Who wants them finer makes them in float32 and calls route_experts.  A token with a NaN
        has NaN logits, which are never chosen: it goes to no expert and comes back as zeros."""
        T = x.shape[0]
        everyone = torch.arange(0, 2 * T, T, dtype=torch.int32, device=x.device)
        bias = self.router_bias.float() if self.router_bias is not None else None   # (the layer may have been cast)
        return route_experts(streamk_grouped(x, self.router[None], everyone), self.chosen, bias=bias, **self.routing)

    def forward(self, x):
        if x.dtype != self.dtype or x.shape[-1] != self.hidden:
            raise ValueError(f"input must be {self.dtype} [..., {self.hidden}], got {x.dtype} {tuple(x.shape)}")
        rows = x.reshape(-1, self.hidden)
        if rows.shape[0] == 0:
            return torch.zeros_like(x)
        if self.weight_format in _QUANTIZED:
            return self._quantized(rows).view(x.shape)
        route = self.route(rows)
        if torch.is_grad_enabled() and (rows.requires_grad or self.up.requires_grad or self.down.requires_grad):
            h = streamk_grouped(dispatch_rows(rows, route), self.up, route.offsets)
            out = streamk_grouped(_ACTIVATIONS[self.activation](h), self.down, route.offsets)
        else:
            h = streamk_grouped(dispatch_rows(rows, route), self.up, route.offsets, activation=self.activation)
            out = streamk_grouped(h, self.down, route.offsets)
        return combine_rows(out, route).view(x.shape)

    @torch.no_grad()   # (inference only, as the other quantised layers)
    def _quantized(self, x):
        quantize = _QUANTIZED[self.weight_format][0]
        route = self.route(x)
        q, scale = quantize(x)
        h = streamk_grouped(dispatch_rows(q, route), self.up, route.offsets, scale_a=dispatch_rows(scale, route), scale_b=self.up_scale,
                            out_dtype=self.dtype, activation=self.activation)
        q, scale = quantize(h)
        return combine_rows(streamk_grouped(q, self.down, route.offsets, scale_a=scale, scale_b=self.down_scale, out_dtype=self.dtype), route)

    def extra_repr(self):
        return (f"hidden={self.hidden}, intermediate={self.intermediate}, experts={self.experts}, chosen={self.chosen}, "
                f"activation={self.activation}, weight_format={self.weight_format}, "
                + ", ".join(f"{name}={value}" for name, value in self.routing.items()) + f", balance={self.router_bias is not None}")
