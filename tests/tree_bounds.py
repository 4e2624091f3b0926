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


def rows_and_bound_by_element(q, k, v, mask, group):
    """The same rows, with a bound for F32 and int8 pools that follows each
    element of K and V, not its row's largest: an element enters as two F16 parts
    with at most 2^-23 of itself left out (the first part is off by at most 2^-11
    of the element, the second by 2^-12 of that), and the product of two second
    parts, at most 2^-22 of the product, is left out.  A row is brought to a
    largest value in [2^14, 2^15), so what F16 cannot hold, at most 2^-25, is
    2^-39 of the row's largest.  With 3 d/16 + 1 truncating additions a score is
    off by at most (3 d/16 + 5) 2^-23 of its sum of |q k|, and by 2^-39 of the
    rows' largest times the other side's sum.  A weight is off by twice that and
    2^-22 of the exponential; the weighted sum adds 24 additions' 2^-23 and the
    parts' 2^-21.  Weight times row scale is below 2^11 and its largest is at
    least 2^3 (a tile's scales within 2^6 of one another, two references rounded
    up), where F16 leaves out 2^-25: 2^-28 of the largest weight times row
    maximum (its power of two at most twice it: 2^-27), of either sign, six
    deviations of sqrt(m) of them.  That largest is taken as no less than 2^-90
    of the largest weight (a little less in fact, so that the sum of unscaled
    weights does not overflow): F16's 2^-25 is then 2^-25 2^-11 2^-90, times
    elements below 2^15: 2^-111, of either sign, again six deviations."""
    import torch
    n, heads, d = q.shape
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    seen = mask.repeat_interleave(group, 0)
    some = seen.any(1)
    for g in range(heads // group):
        qg = q[:, g * group:(g + 1) * group].reshape(n * group, d)
        s = (qg @ k[g].T / np.sqrt(d)).masked_fill(~seen, -torch.inf)
        size = qg.abs() @ k[g].abs().T
        floor = 2.0 ** -39 * (qg.abs().amax(1)[:, None] * k[g].abs().sum(1) + qg.abs().sum(1)[:, None] * k[g].abs().amax(1))
        e = (((3 * -(-d // 16) + 5) * 2.0 ** -23 * size + floor) / np.sqrt(d)).masked_fill(~seen, 0.0).amax(1, keepdim=True)
        w = torch.softmax(s, 1).masked_fill(~some[:, None], 0.0)
        v_seen = v[g].masked_fill(~mask.any(0)[:, None], 0.0)
        row = v_seen.abs().amax(1)
        bound = (w @ v_seen.abs()) * (2 * e + 2.0 ** -22 + 24 * 2.0 ** -23 + 2.0 ** -21) \
            + 2.0 ** -39 * (w @ row)[:, None] \
            + 6 * seen.sum(1, keepdim=True).sqrt() * (2.0 ** -27 * (w * row).amax(1, keepdim=True) + 2.0 ** -111)
        out[:, g * group:(g + 1) * group] = (w @ v_seen).reshape(n, group, d)
        tol[:, g * group:(g + 1) * group] = bound.masked_fill(~some[:, None], 0.0).reshape(n, group, d)
    return out, tol


def check_case(case, bound=rows_and_bound):
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
        want, tol = bound(q, k, v, torch.from_numpy(case.mask[s]).cuda(), case.heads // case.kv_heads)
        off = (got[r, :width].reshape(n, case.heads, case.d) - want).abs()
        assert (off <= tol).all(), (s, off.max().item(), (off - tol).max().item())  # NaN is not below its bound
    assert int(case.dev.keep["status"].item()) == 0
