"""Rotary positions over the C ABI (``cxs_rotary``).

The glue kernel of the extend model rotates whole bf16 heads of 64 in the half
layout. ``Rotary`` covers the other forms: interleaved pairs, part of the
head, frequencies scaled for long contexts, bf16 / fp16 / fp32, strided and
in-place tensors, and the transposed rotation, which is the gradient. The
reference has only the first form (models/tensor_ops.py:14-26).
"""

import math

import torch

from . import _lib

LAYOUTS = {"half": 0, "interleaved": 1}
TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def frequencies(rotary_dim, theta=10000.0, scaling=None):
    """Radians per position of every channel pair (fp64, on the CPU) and the
    factor on the rotated values. ``scaling``:

    - None: theta ** (-2 i / rotary_dim);
    - ``dict(type="linear", factor=s)``: positions divided by s (any s > 0);
    - ``dict(type="ntk", factor=s)``: theta raised so that the slowest pair is
      stretched s times and the fastest is kept;
    - ``dict(type="yarn", factor=s, original=n, fast=32, slow=1)`` (Peng et al.
      2023): pairs that make fewer than ``slow`` turns over ``n`` positions are
      stretched s times, those with more than ``fast`` are kept, a linear ramp
      over the pair index between; values times 0.1 ln(s) + 1 (or ``magnitude``).
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even")
    if not theta > 1:
        raise ValueError("theta must be above 1")
    scaling = dict(scaling or {"type": "none"})
    kind = scaling.pop("type", None)
    fields = {"none": (), "linear": ("factor",), "ntk": ("factor",),
              "yarn": ("factor", "original", "fast", "slow", "magnitude")}
    if kind not in fields:
        raise ValueError(f"unknown rotary scaling {kind!r}")
    unknown = set(scaling) - set(fields[kind])
    if unknown:
        raise ValueError(f"unknown fields of rotary scaling {kind!r}: {sorted(unknown)}")
    factor = float(scaling.get("factor", 1.0))
    if not factor > 0:
        raise ValueError("the scaling factor must be positive")
    if kind == "ntk" and rotary_dim > 2:
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    index = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    f = theta ** (-index / rotary_dim)
    if kind == "linear":
        return f / factor, 1.0
    if kind == "yarn":
        if "original" not in scaling or not scaling["original"] > 0:
            raise ValueError("yarn scaling needs the original context length")
        original = scaling["original"]

        def pair(turns):  # the pair index that makes `turns` turns over `original` positions
            return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))

        low = max(0, math.floor(pair(scaling.get("fast", 32))))
        high = min(rotary_dim - 1, math.ceil(pair(scaling.get("slow", 1))))
        ramp = ((index / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
        magnitude = scaling.get("magnitude", 0.1 * math.log(factor) + 1 if factor > 1 else 1.0)
        return f / factor * ramp + f * (1 - ramp), float(magnitude)
    return f, 1.0


class _Turn(torch.autograd.Function):
    """``Rotary.apply`` under autograd: the gradient is the transposed rotation
    of the outputs' gradients (of those that there are)."""

    @staticmethod
    def forward(ctx, rotary, positions, transpose, q, k):
        ctx.rotary, ctx.transpose = rotary, transpose
        ctx.save_for_backward(positions)
        ctx.set_materialize_grads(False)
        return rotary.apply(q, k, positions, transpose=transpose)

    @staticmethod
    def backward(ctx, q, k):
        # (Gradients of sums are broadcast along the channels.)
        q, k = (g if g is None or g.stride(-1) == 1 else g.contiguous() for g in (q, k))
        if q is not None or k is not None:
            q, k = ctx.rotary.apply(q, k, *ctx.saved_tensors, transpose=not ctx.transpose)
        return None, None, None, q, k


class Rotary:
    """The rotation of one head geometry: ``apply(q, k, positions)``.

    ``steps`` holds each pair's turns per position as a 64-bit fraction, so a
    phase is exact at any position before its sine and cosine are taken."""

    def __init__(self, dim, *, rotary_dim=None, theta=10000.0, layout="half", scaling=None,
                 device="cuda"):
        rotary_dim = dim if rotary_dim is None else rotary_dim
        if dim < 2 or dim % 2 or dim > 512:
            raise ValueError("dim must be even and at most 512")
        if rotary_dim > dim:
            raise ValueError("rotary_dim must be at most dim")
        if layout not in LAYOUTS:
            raise ValueError(f"unknown rotary layout {layout!r}")
        self.dim, self.rotary_dim, self.layout = dim, rotary_dim, layout
        f, self.magnitude = frequencies(rotary_dim, theta, scaling)
        if not (f.isfinite().all() and math.isfinite(self.magnitude)):
            raise ValueError("the scaling's frequencies or magnitude are not finite")
        # Whole turns per position do not matter: at most half a turn is left,
        # whose 2^62-fold fits 64 bits. Doubled twice it wraps modulo one turn,
        # as its product with a position does.
        turns = f / (2 * math.pi)
        steps = ((turns - turns.round()) * 2.0 ** 62).round().to(torch.int64) << 2
        self.steps = steps.to(device)
        self.device = self.steps.device
        self._steps, self._layout = self.steps.data_ptr(), LAYOUTS[layout]

    def _check(self, name, x, dtype):
        """Shape and strides of a [tokens, heads, dim] tensor."""
        shape, stride = x.shape, x.stride()
        if len(shape) != 3 or shape[2] != self.dim or stride[2] != 1:
            raise ValueError(f"{name} must be [tokens, heads, {self.dim}] with contiguous channels")
        if x.dtype != dtype:
            raise ValueError("the tensors must have one type")
        if x.device != self.device:
            raise ValueError(f"{name} must be on {self.device}")
        return shape, stride

    def _side(self, name, x, y, tokens, dtype):
        """(output, input and output address, their strides, heads) of one tensor."""
        if x is None:
            return None, 0, 0, (0, 0, 0, 0), 0
        shape, stride = self._check(name, x, dtype)
        heads = shape[1]
        if shape[0] != tokens:
            raise ValueError("q, k and positions must have as many tokens")
        if y is None:
            y = torch.empty_like(x, memory_format=torch.contiguous_format)
            return y, x.data_ptr(), y.data_ptr(), (stride[0], stride[1], heads * self.dim,
                                                   self.dim), heads
        out_shape, to = self._check(f"out of {name}", y, dtype)
        if out_shape != shape:
            raise ValueError(f"out of {name} must have its shape")
        return y, x.data_ptr(), y.data_ptr(), (stride[0], stride[1], to[0], to[1]), heads

    def apply(self, q, k, positions, *, transpose=False, out=None):
        """Rotated ``(q, k)`` for q [tokens, heads, dim], k [tokens, kv_heads,
        dim] (either may be None) and positions [tokens] int32 or int64, in one
        launch on the current stream. ``transpose`` turns the other way: given
        the gradients of the outputs it returns those of the inputs (and, for
        magnitude 1, undoes the rotation); autograd does so by itself.
        ``out=(q_out, k_out)`` receives the result; each may be its input
        itself, and must not overlap an input in another way. ``out`` has no
        gradient: it is refused for tensors that need one."""
        first = q if q is not None else k
        if first is None:
            raise ValueError("q or k is needed")
        dtype, tokens = first.dtype, first.shape[0]
        if dtype not in TYPES:
            raise ValueError("q and k must be bf16, fp16 or fp32")
        wide = positions.dtype == torch.int64
        if not (wide or positions.dtype == torch.int32) or positions.shape != (tokens,) \
                or positions.device != self.device:
            raise ValueError(f"positions must be [tokens] int32 or int64 on {self.device}")
        if not positions.is_contiguous():
            positions = positions.contiguous()
        needs = first.requires_grad or (k is not None and k.requires_grad)
        if out is None:
            if needs and torch.is_grad_enabled():
                return _Turn.apply(self, positions, bool(transpose), q, k)
            q_out = k_out = None
        else:
            q_out, k_out = out
            if torch.is_grad_enabled() and (needs or any(
                    t is not None and t.requires_grad for t in out)):
                raise ValueError("out cannot receive a result that needs a gradient")
            if (q_out is None) != (q is None) or (k_out is None) != (k is None):
                raise ValueError("out must have a tensor for each of q and k that is given")
        q_out, qp, qo, qs, heads = self._side("q", q, q_out, tokens, dtype)
        k_out, kp, ko, ks, kv_heads = self._side("k", k, k_out, tokens, dtype)
        call = _lib.pack_rotary_call(
            qp, kp, qo, ko, positions.data_ptr(), self._steps, qs[0], qs[1], ks[0], ks[1],
            qs[2], qs[3], ks[2], ks[3], tokens, heads, kv_heads, self.dim, self.rotary_dim,
            self._layout, TYPES[dtype], bool(transpose), wide, self.magnitude)
        _lib.on_device(self.device.index, _lib.packed().cxs_rotary, call)
        if out is not None:
            torch.autograd.graph.increment_version([t for t in out if t is not None])
        return q_out, k_out
