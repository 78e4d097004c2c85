"""Plain 64-bit models of the drafted-token operators, for the GPU tests."""
import math

import torch


def e8m0_rows(x):
    """(values held, scale bytes) of rows x [..., D] in float64, by the definition of the 8-bit cache."""
    x = x.double()
    held, scale = torch.empty_like(x), torch.empty(x.shape[:-1], dtype=torch.uint8, device=x.device)
    flat, out, bytes_ = x.reshape(-1, x.shape[-1]).cpu(), held.view(-1, x.shape[-1]), scale.view(-1)
    for i, row in enumerate(flat):
        largest = max(abs(v) for v in row.tolist()) if torch.isfinite(row).all() else math.inf
        if not math.isfinite(largest):
            out[i], bytes_[i] = math.nan, 255
            continue
        n = -127
        if largest > 0:
            n = max(-127, math.frexp(largest)[1] - 10)
            while largest > 448 * 2.0 ** n:
                n += 1
        y = [v / 2.0 ** n for v in row.tolist()]
        steps = [2.0 ** (max(math.frexp(abs(v))[1] - 1, -6) - 3) for v in y]
        out[i] = torch.tensor([round(v / s) * s * 2.0 ** n for v, s in zip(y, steps)])   # (round: ties to even)
        bytes_[i] = n + 127
    return held, scale


def seen_by(parents, count):
    """[count, count] bool: row i holds node i's ancestors and itself."""
    seen = torch.zeros(count, count, dtype=torch.bool)
    for i in range(count):
        seen[i, i] = True
        if parents[i] >= 0:
            seen[i] |= seen[parents[i]]
    return seen


def tree_attention(q, k, v, prefix, parents):
    """One sequence: q [n,Hq,D], k, v [prefix + n, Hkv, D] in float64; returns (out, mean of |v| under the same
    weights, log of the softmax sums).  What a node does not see is taken out before any arithmetic."""
    n, hq, dim = q.shape
    group = hq // k.shape[1]
    seen = torch.cat([torch.ones(n, prefix, dtype=torch.bool), seen_by(parents, n)], 1).to(q.device)
    out, mean, lse = torch.empty_like(q), torch.empty_like(q), torch.empty(n, hq, dtype=q.dtype, device=q.device)
    for i in range(n):
        kk, vv = k[seen[i]].repeat_interleave(group, 1), v[seen[i]].repeat_interleave(group, 1)
        s = torch.einsum("hd,thd->ht", q[i], kk) / math.sqrt(dim)
        w = torch.softmax(s, -1)
        out[i], mean[i] = torch.einsum("ht,thd->hd", w, vv), torch.einsum("ht,thd->hd", w, vv.abs())
        lse[i] = torch.logsumexp(s, -1)
    return out, mean, lse


def verify(p, tokens, u, u_last, parents, count, q=None):
    """One sequence, walked node by node; p [n + 1][V], q [n][V] or None as lists of floats."""
    path, node, tree = [], -1, parents is not None
    tried, left, rest = [], 1.0, list(p[0])
    i = 0
    while i < count:
        parent = parents[i] if tree else i - 1
        x = tokens[i]
        valid = 0 <= x < len(p[0]) and -1 <= parent < i
        if parent == node:
            given = q is None
            if tree:
                good = valid and x not in tried and u[i] * left < p[node + 1][x]
            else:
                good = valid and u[i] * (1.0 if given else q[i][x]) < p[node + 1][x]
            if good:
                path.append(i)
                node, tried, left, rest = i, [], 1.0, list(p[i + 1])
            elif tree:
                if valid:
                    left -= 0.0 if x in tried else p[node + 1][x]
                    tried.append(x)
                    rest[x] = 0.0
            else:
                if given:
                    if valid:
                        rest[x] = 0.0
                else:
                    rest = [max(a - b, 0.0) for a, b in zip(p[node + 1], q[i])]
                break
        elif not tree:
            break
        i += 1
    for row in (rest, p[node + 1]):
        total = math.fsum(row) if not any(math.isnan(z) for z in row) else math.nan
        if total > 0:
            break
    drawn = -1
    if total > 0 and math.isfinite(total):
        run, drawn = 0.0, None
        for x, w in enumerate(row):
            run += w
            if run > u_last * total:
                drawn = x
                break
        if drawn is None:
            drawn = max(x for x, w in enumerate(row) if w > 0)
    n = len(tokens)
    return len(path), path + [-1] * (n - len(path)), [tokens[j] for j in path] + [drawn] + [-1] * (n - len(path))
