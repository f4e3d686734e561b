"""A paged cache and attention over it, stated plainly on the CPU in 64 bits: what the tests of the kernels compare with."""
import numpy as np
import torch

NO_PAGE = -1


def tables(cached, new, table, free, page_size, tokens):
    """(page table, slots, row starts, counts) as lists, by the definition."""
    table, free = [list(row) for row in table], list(free)
    slots, starts, taken, missing = [], [0], 0, 0
    for r, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        width = len(table[r])
        held, want = min(width, -(-c // page_size)), min(width, -(-(c + n) // page_size))
        for j in range(held, width):
            table[r][j] = NO_PAGE
            if j < want:
                if taken < len(free):
                    table[r][j] = free[taken]
                    taken += 1
                else:
                    missing += 1
        for p in range(c, c + n):
            page = table[r][p // page_size] if p // page_size < width else NO_PAGE
            slots.append(page * page_size + p % page_size if page >= 0 else -1)
        starts.append(starts[-1] + n)
    return table, (slots + [-1] * tokens)[:tokens], [min(s, tokens) for s in starts], [taken, missing]


def attention(rows, keys, values, table, cached, starts, heads, head_dim, page_size, query_column=0, scale=None, window=0):
    """(out, bound) [tokens, heads * head_dim] in 64 bits.  keys, values: [pages, kv_heads, page_size, head_dim] float64.

    bound: how far a kernel may be off that adds up in fp32, rounds the probabilities and the result to bf16.  With the weights w_j
    of a row, A = sum_j w_j |v_j| element by element and e the largest error of a score (head_dim + 2 roundings of its terms in
    fp32, and the exponential's own 2^-21):  2^-9 |out| for the result's rounding (half of what that
    can take: bf16 has 8 significant bits), 2^-8 A for that of the probabilities and for their sum in
    the denominator, 2 e A for the scores (numerator and denominator), and as much again as 2^-20 A for the sums."""
    kv_heads, pages = keys.shape[1], keys.shape[0]
    scale = head_dim ** -0.5 if scale is None else scale
    tokens = rows.shape[0]
    out, bound = torch.zeros(tokens, heads, head_dim, dtype=torch.float64), torch.zeros(tokens, heads, head_dim, dtype=torch.float64)
    for r, c in enumerate(cached):
        for t in range(starts[r], starts[r + 1]):
            p = c + t - starts[r]
            first = max(0, p + 1 - window) if window else 0
            where = [(table[r][j // page_size], j % page_size) for j in range(first, p + 1) if j // page_size < len(table[r])]
            where = [(page, at) for page, at in where if 0 <= page < pages]
            if not where:
                continue
            page, at = (torch.tensor(x) for x in zip(*where))
            k, v = keys[page, :, at].transpose(0, 1), values[page, :, at].transpose(0, 1)              # [kv_heads, seen, head_dim]
            q = rows[t, query_column:query_column + heads * head_dim].double().view(kv_heads, heads // kv_heads, head_dim)
            scores = q @ k.transpose(1, 2) * scale
            weights = torch.softmax(scores, dim=-1)
            o, a = weights @ v, weights @ v.abs()
            e = (head_dim + 2) * 2.0 ** -23 * abs(scale) * (q.abs() @ k.abs().transpose(1, 2)).amax(dim=-1, keepdim=True) + 2.0 ** -21
            out[t] = o.reshape(heads, head_dim)
            bound[t] = (2.0 ** -9 * o.abs() + (2.0 ** -8 + 2 * e + 2.0 ** -20) * a + 1e-30).reshape(heads, head_dim)
    return out.flatten(1), bound.flatten(1)


def bfloat8_b(oracle, x):
    """What a BFLOAT8_B tensor of x [..., H, W] (whole tiles) holds, float32, through the oracle's packer."""
    a = np.ascontiguousarray(x.float().numpy()).reshape(-1, *x.shape[-2:])
    return torch.from_numpy(oracle.to_torch_bfp_tiles(3, oracle.from_torch_bfp_tiles(3, a), a.shape).reshape(x.shape))
