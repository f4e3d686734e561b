"""Positions, sinks and pages that change hands around a paged cache, stated plainly on the CPU in 64 bits: what the tests of the kernels compare with."""
import torch

NO_PAGE = -1


def owners(cached, starts, tokens):
    """(request, position) of every row, None for rows of no request; a start below an earlier one is read as that one."""
    out, taken = [None] * tokens, min(max(starts[0], 0), tokens)
    for r, c in enumerate(cached):
        end = max(taken, min(max(starts[r + 1], 0), tokens))
        for t in range(taken, end):
            out[t] = (r, max(c, 0) + t - taken)
        taken = end
    return out


def rotate(rows, positions, heads, head_dim, frequencies, interleaved=False, norm=None, epsilon=0.0, magnitude=1.0):
    """(out, bound) [tokens, heads, head_dim] in 64 bits: rows [tokens, heads * head_dim], positions as owners() gives them.  Rows without one are zeros.

    bound: how far a kernel may be off before its result is rounded.  With a, b the elements that go into a result and m the magnitude,
      |a| + |b| times m times
        2^-21        sine and cosine (2^-22.9 off at most, over all multiples of 2^-24 of a turn) and the rounding of the turn to 24 bits, 2 pi 2^-26
        p f 2^-49    the turn in 64 bits: the constant 1 / 2 pi, its product with f and that with p, 2^-53 p f / 2 pi each, is 2 pi times that of an angle;
                     here and there, and as much again for what cos and sin below are given
        2^-21        the product with m, two products and a sum, 2^-24 each
        (D / 2 + 8) 2^-24    where there is a norm: half of what D products and sums can be off, and a reciprocal root and two products
    """
    tokens, pairs = rows.shape[0], frequencies.numel()
    x = rows.double().view(tokens, heads, head_dim)
    if norm is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + epsilon) * norm.double()
    p = torch.tensor([0 if o is None else o[1] for o in positions], dtype=torch.float64)
    angle = (p[:, None] * frequencies.double())[:, None]
    cos, sin = torch.cos(angle), torch.sin(angle)
    if interleaved:
        first, second = 2 * torch.arange(pairs), 2 * torch.arange(pairs) + 1
    else:
        first, second = torch.arange(pairs), torch.arange(pairs) + pairs
    out, size = x.clone(), x.abs()
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = magnitude * (a * cos - b * sin), magnitude * (b * cos + a * sin)
    both = abs(magnitude) * (a.abs() + b.abs())
    relative = 2.0 ** -20 + angle.abs() * 2.0 ** -49
    bound = torch.zeros_like(x)
    bound[..., first] = bound[..., second] = both * relative
    size[..., first] = size[..., second] = both
    if norm is not None:
        bound = bound + size * (head_dim / 2 + 8) * 2.0 ** -24
    there = torch.tensor([o is not None for o in positions])[:, None, None]
    return torch.where(there, out, 0.0), torch.where(there, bound, 0.0)


def as_bfloat16(out, bound):
    """The bound of a result that is rounded to bf16: half a step of what it rounds, 2^-8 of it."""
    return bound + 2.0 ** -8 * (out.abs() + bound) + 1e-38


def as_bfloat8_b(out, bound):
    """(values, bound) of a result [.., 16 n] that is packed 16 neighbours at a time: a step is 2^-6 of the power of two at or below the largest one; rounding
    takes half of it, and the largest code, 127, as much as a whole one.  Where the error can bring the largest one over a power of two, the step is the larger one."""
    x, e = out.unflatten(-1, (-1, 16)), bound.unflatten(-1, (-1, 16))
    top = (x.abs() + e).amax(-1, keepdim=True).clamp(min=2.0 ** -100)
    step = 2.0 ** (torch.floor(torch.log2(top)) - 6)
    over = (x.abs() + e - 127 * step).clamp(min=0.0)
    return (e + torch.maximum(step / 2, over)).flatten(-2)


def attention(rows, keys, values, table, cached, starts, heads, head_dim, page_size, query_column=0, scale=None, window=0, sinks=0):
    """(out, bound) [tokens, heads * head_dim] in 64 bits.  keys, values: [pages, kv_heads, page_size, head_dim] float64.

    bound: scores and sums in fp32, weights and result rounded to bf16.  With the weights w_j of a row, A = sum_j w_j |v_j| and e the largest error of a score
    (head_dim + 2 roundings of its terms, and the exponential's own 2^-21): 2^-8 |out| for the result, 2^-8 A for the weights in numerator and
    denominator, 2 e A for the scores in both, 2^-20 A for the sums."""
    kv_heads, pages = keys.shape[1], keys.shape[0]
    scale = head_dim ** -0.5 if scale is None else scale
    tokens = rows.shape[0]
    out, bound = torch.zeros(tokens, heads, head_dim, dtype=torch.float64), torch.zeros(tokens, heads, head_dim, dtype=torch.float64)
    for t, owner in enumerate(owners(cached, starts, tokens)):
        if owner is None:
            continue
        r, p = owner
        reach = min(p + 1, len(table[r]) * page_size)
        seen = [j for j in range(reach) if not window or j > p - window or j < sinks]
        where = [(table[r][j // page_size], j % page_size) for j in seen]
        where = [(page, at) for page, at in where if 0 <= page < pages]
        if not where:
            continue
        page, at = (torch.tensor(x) for x in zip(*where))
        k, v = keys[page, :, at].transpose(0, 1), values[page, :, at].transpose(0, 1)
        q = rows[t, query_column:query_column + heads * head_dim].double().view(kv_heads, heads // kv_heads, head_dim)
        weights = torch.softmax(q @ k.transpose(1, 2) * scale, dim=-1)
        o, a = weights @ v, weights @ v.abs()
        e = (head_dim + 2) * 2.0 ** -23 * abs(scale) * (q.abs() @ k.abs().transpose(1, 2)).amax(dim=-1, keepdim=True) + 2.0 ** -21
        out[t] = o.reshape(heads, head_dim)
        bound[t] = (2.0 ** -8 * o.abs() + (2.0 ** -8 + 2 * e + 2.0 ** -20) * a + 1e-30).reshape(heads, head_dim)
    return out.flatten(1), bound.flatten(1)


def fork(table, lengths, parents, free, page_size):
    """(page table, lengths, sources, targets, counts) as lists, by the definition."""
    free, seen, taken, missing = list(free), set(), 0, 0
    rows, out, sources, targets = [], [], [], []
    for parent in parents:
        width = len(table[0]) if table else 0
        row, n, source, target = [NO_PAGE] * width, 0, NO_PAGE, NO_PAGE
        if 0 <= parent < len(table):
            n = max(lengths[parent], 0)
            row = [page if j * page_size < n else NO_PAGE for j, page in enumerate(table[parent])]
            begun = n // page_size
            if parent in seen and n % page_size and begun < width and row[begun] >= 0:
                if taken < len(free):
                    if free[taken] >= 0:
                        source, target = row[begun], free[taken]
                    row[begun] = free[taken]
                    taken += 1
                else:
                    row[begun] = NO_PAGE
                    missing += 1
            seen.add(parent)
        rows.append(row)
        out.append(n)
        sources.append(source)
        targets.append(target)
    return rows, out, sources, targets, [taken, missing]


def release(table, lengths, page_size, pages, window=0, sinks=0):
    """(page table, free pages, counts) as lists, by the definition."""
    rows, used = [], set()
    for row, n in zip(table, lengths):
        n, kept = max(n, 0), []
        for j, page in enumerate(row):
            tokens = range(j * page_size, min(n, (j + 1) * page_size))
            # what a token at n or later can see: the window of the one at n, and the sinks; the page's own tokens up to its end
            needed = len(tokens) and (not window or (j + 1) * page_size - 1 > n - window or j * page_size < sinks)
            kept.append(page if needed and 0 <= page < pages else NO_PAGE)
            if kept[-1] >= 0:
                used.add(page)
        rows.append(kept)
    free = [page for page in range(pages) if page not in used]
    return rows, free + [NO_PAGE] * len(used), [len(free), len(used)]
