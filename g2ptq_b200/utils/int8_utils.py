"""8-bit linears: what runs a weight that ``fasterquant`` or a ``WeightQuantizer``
quantized to int8 codes with one scale per channel.

Activations are quantized per token as they arrive (the reference's per-token
symmetric ``ActQuantizer``, utils/quant_utils.py:167-338, which only emulates it
in the model's type); the codes are multiplied as integers and the sums scaled
per token and per channel.  Inference only: nothing here records gradients, and
inputs that require one are refused under grad mode (``RuntimeError``).
"""

import torch

from .. import ops


def _int8_rows(codes):
    """``codes`` with rows padded with zeros to 16-byte boundaries."""
    *lead, cols = codes.shape
    out = torch.zeros(*lead, ops.int8_row_stride(cols), dtype=torch.int8, device=codes.device)
    out[..., :cols].copy_(codes)
    return out


def _plain_rows(x):
    """``x [M, K]`` with unit column stride and rows that do not overlap (a broadcast
    tensor's lie on top of each other)."""
    if x.is_contiguous():
        return x
    (rows, cols), (step, unit) = x.shape, x.stride()
    return x.contiguous() if (cols > 1 and unit != 1) or (rows > 1 and step < cols) else x


def int8_linear(x, codes, scale, bias=None):
    """``x @ (scale[:, None] * codes).T + bias`` with ``x [..., K]`` quantized per
    token: int8 ``codes [N, K]``, fp32 ``scale [N]`` and ``bias [N]``.  The result
    has ``x``'s type."""
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    y = ops.int8_linear(_plain_rows(x2), codes, scale, bias)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], y.shape[1])


def int8_experts(x, codes, scale, offsets):
    """``int8_linear`` of rows sorted by expert (``moe_utils.dispatch``): rows
    ``offsets[e]`` to ``offsets[e + 1] - 1`` of ``x [R, K]`` through expert
    ``e``'s ``codes [E, N, K]`` and ``scale [E, N]``.  Rows behind the last
    expert's give zeros."""
    return ops.int8_linear_grouped(_plain_rows(x) if x.dim() == 2 else x, codes, scale, offsets)


def weight_codes(weight, quantizer):
    """int8 codes ``[N, K]`` and fp32 scales ``[N]`` of ``weight`` on the grid of a
    ready ``WeightQuantizer``: symmetric, one scale per channel."""
    if not quantizer.ready() or not quantizer.sym or quantizer.weight_groupsize > 0:
        raise ValueError("8-bit linears need a ready symmetric quantizer with one scale per "
                         "channel (no groups)")
    if quantizer.bits > 8:
        raise ValueError(f"codes of {quantizer.bits} bits do not fit int8")
    if quantizer.scale.numel() not in (1, weight.shape[0]):
        raise ValueError(f"the quantizer has {quantizer.scale.numel()} scales for "
                         f"{weight.shape[0]} channels (of a layer-batched object take each "
                         "layer's rows with merge_group_quantizers)")
    _, q, scale = quantizer.fake_quantize(weight)
    scale = scale.reshape(-1).float()
    if scale.numel() == 1:
        scale = scale.expand(weight.shape[0])
    return q.to(torch.int8), scale.contiguous()


class _Int8Weight(torch.nn.Module):
    """int8 codes and channel scales.  The buffer ``rows`` holds the padded rows (so
    that moving or copying the module keeps their alignment), ``codes`` is the
    view of the columns.  Converting the module (``model.to(torch.bfloat16)``,
    ``.half()``) moves the buffers and leaves their types and values: they are what
    the quantization chose, whatever type the activations have."""

    def __init__(self, codes, scale):
        super().__init__()
        self.out_features, self.in_features = codes.shape[-2:]
        self.register_buffer("rows", _int8_rows(codes))
        self.register_buffer("scale", scale.detach().float().contiguous())

    def _apply(self, fn, *args, **kwargs):
        kept = dict(self._buffers)
        super()._apply(fn, *args, **kwargs)
        for name, old in kept.items():
            new = self._buffers[name]
            if old is not None and new.dtype != old.dtype:
                self._buffers[name] = old.to(new.device)
        return self

    @property
    def codes(self):
        rows = self.rows
        return rows if rows.shape[-1] == self.in_features else rows[..., :self.in_features]


class Int8Linear(_Int8Weight):
    """A linear that holds int8 codes ``[N, K]`` and channel scales ``[N]``."""

    def __init__(self, codes, scale, bias=None):
        super().__init__(codes, scale.reshape(-1))
        self.register_buffer("bias", None if bias is None else bias.detach().float().contiguous())

    @classmethod
    def from_linear(cls, linear, quantizer):
        """The codes of ``linear.weight`` on ``quantizer``'s grid: after
        ``fasterquant`` with that quantizer (``obj.quantizer[0]`` for
        ``groupsize`` -1), the codes it chose."""
        codes, scale = weight_codes(linear.weight.data, quantizer)
        return cls(codes, scale, linear.bias)

    def forward(self, x):
        return int8_linear(x, self.codes, self.scale, self.bias)


class Int8Experts(_Int8Weight):
    """The same projection of every expert of an MoE layer, stacked: codes
    ``[E, N, K]`` and scales ``[E, N]``."""

    @classmethod
    def from_linears(cls, linears, quantizers):
        """One quantizer per linear.  Linears with a bias are refused: the grouped
        product has none."""
        linears = list(linears)
        if any(getattr(lin, "bias", None) is not None for lin in linears):
            raise ValueError("8-bit experts have no bias; a linear that has one needs Int8Linear")
        pairs = [weight_codes(lin.weight.data, q)
                 for lin, q in zip(linears, quantizers, strict=True)]
        return cls(torch.stack([c for c, _ in pairs]), torch.stack([s for _, s in pairs]))

    def forward(self, rows, offsets):
        return int8_experts(rows, self.codes, self.scale, offsets)
