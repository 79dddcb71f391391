"""Drawing tokens from logits over the C ABI (``cxs_sample``).

Random numbers are given by the caller, so a run can be repeated, and so can a
captured graph whose numbers are refilled. No counterpart in the reference,
whose models score candidates and draw none. No gradient passes through.
"""

import math

import torch

from . import _lib

TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _setting(name, value, dtype, rows, device):
    """(pointer or 0, value for all rows) of a number or a [rows] tensor."""
    if not isinstance(value, torch.Tensor):
        return 0, value
    if value.shape != (rows,) or value.dtype != dtype or not value.is_contiguous() \
            or value.device != device:
        raise ValueError(f"{name} must be a number or [{rows}] {dtype}, contiguous, on {device}")
    return value.data_ptr(), 0


def sample(logits, uniforms, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
           return_logprobs=False):
    """Tokens (int64, the shape of ``uniforms``) drawn from ``logits [rows,
    vocab]`` (bf16, fp16 or fp32; rows may lie apart) with ``uniforms [rows]`` or
    ``[rows, draws]`` (fp32 or fp64 in [0, 1)).

    Tokens are ordered by logit, equal ones by index. Of softmax(logits /
    temperature), kept are at most the first ``top_k`` (0: all), those at least
    ``min_p`` times as likely as the first, and of what these leave the tokens
    before which less than ``top_p`` of the mass lies; the token is where the
    kept mass, summed by index, passes ``uniforms`` times the whole. Temperature
    0 takes the first token. Each setting is a number (fp32 when it is used) or
    a [rows] tensor (``top_k`` int32, the others fp32). Logits of -infinity or
    NaN are never drawn; a row with no other, or with a setting out of range,
    gets -1.

    With ``return_logprobs`` also the tokens' log softmax(logits), fp32, with no
    temperature and nothing cut (-infinity where the token is -1)."""
    device, shape, size, strides = logits.device, uniforms.shape, logits.shape, logits.stride()
    if len(size) != 2 or logits.dtype not in TYPES or size[1] < 1 \
            or (strides[1] != 1 and size[1] > 1):
        raise ValueError("logits must be [rows, vocab] in bf16, fp16 or fp32 with contiguous rows")
    rows, vocab = size
    if len(shape) not in (1, 2) or shape[0] != rows \
            or uniforms.dtype not in (torch.float32, torch.float64) \
            or not uniforms.is_contiguous() or uniforms.device != device:
        raise ValueError(f"uniforms must be [{rows}] or [{rows}, draws] in fp32 or fp64, "
                         f"contiguous, on {device}")
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("sampling has no gradient: give detached logits")
    heat_at, heat = _setting("temperature", temperature, torch.float32, rows, device)
    k_at, k = _setting("top_k", top_k, torch.int32, rows, device)
    p_at, p = _setting("top_p", top_p, torch.float32, rows, device)
    min_at, least = _setting("min_p", min_p, torch.float32, rows, device)
    if not 0 <= heat < math.inf or not 0 <= k or not p >= 0 or not 0 <= least <= 1:
        raise ValueError("temperature, top_k and top_p must not be negative, min_p be 0 .. 1")
    tokens = uniforms.new_empty(shape, dtype=torch.int64)
    logprobs = uniforms.new_empty(shape, dtype=torch.float32) if return_logprobs else None
    call = _lib.pack_sample_call(
        logits.data_ptr(), uniforms.data_ptr(), tokens.data_ptr(),
        0 if logprobs is None else logprobs.data_ptr(), heat_at, k_at, p_at, min_at,
        strides[0], rows, vocab, 1 if len(shape) == 1 else shape[1], TYPES[logits.dtype],
        uniforms.dtype == torch.float64, heat, min(int(k), vocab), p, least)
    _lib.on_device(device.index, _lib.packed().cxs_sample, call)
    return (tokens, logprobs) if return_logprobs else tokens
