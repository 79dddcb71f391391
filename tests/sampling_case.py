"""Drawing a token from one row of logits, in fp64, step by step."""

import numpy


def draw(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token for each of `u`, log softmax of `x`): numpy fp64; -1 where nothing
    can be drawn. Settings are taken in fp32."""
    x = numpy.asarray(x, dtype=numpy.float64)
    x = numpy.where(numpy.isnan(x), -numpy.inf, x)
    temperature, top_p, min_p = (float(numpy.float32(v)) for v in (temperature, top_p, min_p))
    wrong = not 0 <= temperature < numpy.inf or top_k < 0 or not top_p >= 0 or not 0 <= min_p <= 1
    top = x.max()
    if wrong or top == -numpy.inf:
        return numpy.full(len(u), -1), numpy.full(len(x), -numpy.inf)
    with numpy.errstate(invalid="ignore", divide="ignore"):
        far = numpy.where(x == top, 0.0, x - top)
        logprobs = far - numpy.log(numpy.exp(far).sum())
        order = numpy.lexsort((numpy.arange(len(x)), -x))
        order = order[x[order] > -numpy.inf]
        if temperature == 0 or top_k == 1:
            return numpy.full(len(u), order[0]), logprobs
        if top_k:
            order = order[:top_k]
        if min_p > 0:
            order = order[far[order] >= temperature * numpy.log(min_p)]
        w = numpy.exp(far[order] / temperature)
        if top_p < 1:
            before = numpy.cumsum(w) - w
            n = max(1, int((before < top_p * w.sum()).sum()))
            order, w = order[:n], w[:n]
    back = numpy.argsort(order)
    order, w = order[back], w[back]
    sums = numpy.cumsum(w)
    u = numpy.clip(numpy.nan_to_num(numpy.asarray(u, dtype=numpy.float64), nan=0.0), 0, 1)
    at = numpy.searchsorted(sums, u * sums[-1], side="right")
    last = numpy.flatnonzero(w)[-1]                 # (u of 1: the last that can be drawn)
    return order[numpy.minimum(at, last)], logprobs
