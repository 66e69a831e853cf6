"""Plain 64-bit evaluation of the cache operators, sequence by sequence, and bounds on what the kernels may be off by."""
import math

import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}   # half a step, relative


def rotate(x, pos, rotary, base=10000.0, interleaved=False, inv_freq=None):
    """x [n, heads, dim] float64 turned by pos [n] * frequency."""
    if not rotary:
        return x
    f = torch.as_tensor(inv_freq, dtype=torch.float64) if inv_freq is not None else \
        base ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    ang = pos.double()[:, None, None] * f
    y = x.clone()
    a = slice(0, rotary, 2) if interleaved else slice(0, rotary // 2)
    b = slice(1, rotary, 2) if interleaved else slice(rotary // 2, rotary)
    y[..., a] = x[..., a] * ang.cos() - x[..., b] * ang.sin()
    y[..., b] = x[..., a] * ang.sin() + x[..., b] * ang.cos()
    return y


def spans(lens, starts, tokens):
    """(first row, new tokens, length) per sequence."""
    if starts is None:
        return [(i, 1, int(n)) for i, n in enumerate(lens)]
    out = []
    for i, n in enumerate(lens):
        a, b = max(0, int(starts[i])), min(tokens, int(starts[i + 1]))
        out.append((a, max(0, b - a), int(n)))
    return out


def slots(table_row, page, n_pages, cap, lo, hi):
    """(position, page, slot) of the positions in [lo, hi) that have a page."""
    got = []
    for p in range(max(0, lo), min(hi, cap)):
        pg = int(table_row[p // page])
        if 0 <= pg < n_pages:
            got.append((p, pg, p % page))
    return got


def append(kc, vc, table, lens, starts, k, v, rope):
    """(k cache, v cache, bound of k, written) in float64; the caches hold what they held elsewhere."""
    n_pages, heads, page, dim = kc.shape
    kx, vx = kc.double().cpu().clone(), vc.double().cpu().clone()
    bound = torch.zeros_like(kx)
    written = torch.zeros(kx.shape, dtype=torch.bool)
    tokens = k.shape[0]
    k, v = k.double().cpu().reshape(tokens, heads, dim), v.double().cpu().reshape(tokens, heads, dim)
    for i, (first, n, length) in enumerate(spans(lens, starts, tokens)):
        for j in range(n):
            pos = length - n + j
            for _, pg, sl in slots(table[i], page, n_pages, table.shape[1] * page, pos, pos + 1):
                x = k[first + j][None]
                kx[pg, :, sl] = rotate(x, torch.tensor([pos]), **rope)[0]
                vx[pg, :, sl] = v[first + j]
                # a rotated element is two products: cos and sin are off by at most 2^-22 (half a step of the angle's rest,
                # 2^-26 of a turn, plus two ulps of the function), each product and the sum by half a step
                mag = x.abs() + rotate_partner(x, **rope).abs()
                bound[pg, :, sl] = mag[0] * 2.0 ** -21
                written[pg, :, sl] = True
    return kx, vx, bound, written


def rotate_partner(x, rotary, interleaved=False, **_):
    y = torch.zeros_like(x)
    if rotary:
        a = slice(0, rotary, 2) if interleaved else slice(0, rotary // 2)
        b = slice(1, rotary, 2) if interleaved else slice(rotary // 2, rotary)
        y[..., a], y[..., b] = x[..., b], x[..., a]
    return y


def attend(kc, vc, table, lens, starts, q, heads, rope, scale=None, window=0, out_dtype=torch.float32):
    """(output, bound, row belongs to a sequence) in float64."""
    n_pages, hk, page, dim = kc.shape
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    tokens, group = q.shape[0], heads // hk
    u = U[kc.dtype]
    kc, vc = kc.double().cpu(), vc.double().cpu()
    q = q.double().cpu().reshape(tokens, heads, dim)
    out = torch.zeros((tokens, heads, dim), dtype=torch.float64)
    bound = torch.zeros_like(out)
    mine = torch.zeros(tokens, dtype=torch.bool)
    for i, (first, n, length) in enumerate(spans(lens, starts, tokens)):
        if n == 0:
            continue
        mine[first:first + n] = True
        pos = torch.arange(length - n, length)
        qr = rotate(q[first:first + n], pos, **rope) * scale
        got = slots(table[i], page, n_pages, table.shape[1] * page, 0, length)
        if not got:
            continue
        at = torch.tensor([g[0] for g in got])
        pg, sl = torch.tensor([g[1] for g in got]), torch.tensor([g[2] for g in got])
        seen = at[None] <= pos[:, None]
        if window:
            seen &= at[None] > pos[:, None] - window
        for h in range(heads):
            k, v = kc[pg, h // group, sl], vc[pg, h // group, sl]
            for j in range(n):                      # row by row: what a row does not see never meets it
                m = seen[j]
                if not m.any():
                    continue
                s = k[m] @ qr[j, h]
                p = torch.softmax(s, 0)
                out[first + j, h] = p @ v[m]
                # a score is a sum of dim products: the operands' roundings (rotation 2^-21, and 2^-22 for what the split of
                # q into 16-bit parts leaves), and at most dim / 8 accumulations of partial sums below A cut off at 2^-23
                A = float((k[m].abs() @ qr[j, h].abs()).max())
                ds = A * (2.0 ** -21 + 2.0 ** -22 + dim / 8 * 2.0 ** -23) + float(s.abs().max()) * 2.0 ** -23
                W = p @ v[m].abs()
                if out_dtype == torch.bfloat16:
                    ds += A * u                     # q may be rounded to the cache's type once
                rel = math.expm1(2 * ds) + (int(m.sum()) / 8 + 16) * 2.0 ** -23 + 2.0 ** -20
                if out_dtype == torch.bfloat16:
                    rel += u                        # and so may the weights
                b = W * rel
                if out_dtype == torch.bfloat16:
                    b = b + (out[first + j, h].abs() + b) * U[torch.bfloat16]
                bound[first + j, h] = b + 1e-30
    return out.reshape(tokens, -1), bound.reshape(tokens, -1), mine


def rows_off(got, want, dim, skip=None):
    """How far each (token, head) row is off, relative to its length; element `skip` left out.  The bound above adds up what all
    roundings could do together, which for a bf16 result over many keys is more than the result: whole key tiles could be missing
    inside it.  The roundings are independent (result, weights and q: each at most 2^-8 of its terms, 2^-8 / sqrt(3) in the mean
    square), together at most 2^-8 of a row of values around 0; a test allows 2^-7."""
    keep = [i for i in range(dim) if i != skip]
    d, w = ((x.double().cpu().reshape(-1, dim)[:, keep]) for x in (got - want, want))
    return d.norm(dim=1) / w.norm(dim=1).clamp(min=1e-12)
