"""Users that have their first tokens in common, in pages."""

import torch

from cache8_case import offsets_of, paged


def family(groups, **kw):
    """Cache and call of ``groups``: a list of (common tokens, [(own tokens before
    the new ones, new tokens) of each user]). Full pages of the common tokens are
    the first user's in every row; of a partly filled one each user has a copy
    of those slots. What nobody wrote holds NaN codes."""
    lengths, new, edges, shared = [], [], [0], []
    for common, users in groups:
        lengths += [common + own + n for own, n in users]
        new += [n for _, n in users]
        edges.append(len(lengths))
        shared.append(common)
    codes, scales, table = paged(lengths, **kw)
    size, raw = codes.shape[3], codes.view(torch.uint8)
    for common, low, high in zip(shared, edges, edges[1:]):
        full, fill = common // size, common % size
        for b in range(low + 1, high):
            table[b, :full] = table[low, :full]
            if fill:
                source, target = table[low, full].item(), table[b, full].item()
                raw[target, :, :, :fill] = raw[source, :, :, :fill]
                scales[target] = scales[source]

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=codes.device)

    return dict(codes=codes, scales=scales, table=table, lengths=lengths, new=new,
                call=(table, ints(lengths), offsets_of(new), ints(edges), ints(shared)))
