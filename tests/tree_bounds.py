"""The 64-bit form of tree attention for larger batches than
tests/tree_cases.py's loops take: the same rows and the same rounding bound,
a KV head of a sequence at a time on the GPU."""

import numpy as np


def rows_and_bound(q, k, v, mask, group):
    """tests/tree_cases.py ``attention`` (without its split) for torch arrays in
    64 bits: q [n, heads, d], k and v [kv_heads, m, d], mask [n, m]."""
    import torch
    n, heads, d = q.shape
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    seen = mask.repeat_interleave(group, 0)  # vectors of a KV head: node, then head
    some = seen.any(1)
    for g in range(heads // group):
        qg = q[:, g * group:(g + 1) * group].reshape(n * group, d)
        s = (qg @ k[g].T / np.sqrt(d)).masked_fill(~seen, -torch.inf)
        size = (qg.abs() @ k[g].abs().T / np.sqrt(d)).masked_fill(~seen, 0.0)
        w = torch.softmax(s, 1).masked_fill(~some[:, None], 0.0)
        e = (2 * -(-d // 16) + 1) * 2.0 ** -23 * size.amax(1, keepdim=True)
        top = torch.stack([v[g].abs().masked_fill(~row[:, None], 0.0).amax(0) for row in mask]).repeat_interleave(group, 0)
        bound = (w @ v[g].abs()) * (2 * e + 2.0 ** -22 + 24 * 2.0 ** -23) \
            + 6 * seen.sum(1, keepdim=True).sqrt() * 2.0 ** -25 * top + 1e-30
        out[:, g * group:(g + 1) * group] = (w @ v[g]).reshape(n, group, d)
        tol[:, g * group:(g + 1) * group] = bound.masked_fill(~some[:, None], 0.0).reshape(n, group, d)
    return out, tol


def check_case(case):
    """A tree_cases.AttentionCase that has run: every row within its bound, rows
    behind the last sequence as they were, no status bit."""
    import torch
    width, total = case.heads * case.d, case.total
    got = case.dev.keep["out"].double()
    assert torch.equal(case.dev.keep["out"][total:].cpu(), torch.from_numpy(case.out[total:]))
    for s, n in enumerate(case.nodes):
        if not n:
            continue
        r = slice(int(case.cu[s]), int(case.cu[s + 1]))
        q = torch.from_numpy(case.q[r, :width].astype(np.float64)).cuda().reshape(n, case.heads, case.d)
        k, v = (torch.from_numpy(np.ascontiguousarray(x[s])).cuda() for x in (case.k, case.v))
        want, tol = rows_and_bound(q, k, v, torch.from_numpy(case.mask[s]).cuda(), case.heads // case.kv_heads)
        off = (got[r, :width].reshape(n, case.heads, case.d) - want).abs()
        assert (off <= tol).all(), (s, off.max().item(), (off - tol).max().item())  # NaN is not below its bound
    assert int(case.dev.keep["status"].item()) == 0
