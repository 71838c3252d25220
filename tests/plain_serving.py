"""Packed and paged attention, 8-bit caches and sampling in 64 bits, sequence by sequence and head by head, with bounds of what the
kernels' roundings may change (``u`` is half a step of the 16-bit type: 2^-8 for bf16, 2^-11 for fp16)."""
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALL = 2.0 ** -13          # 32-bit scores, exponentials and sums: 128 terms of 2^-24 each, scores up to 32 in an exponent, twice


def starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def visible(n, m, window, device):
    ahead = torch.arange(m, device=device)[None] - (torch.arange(n, device=device)[:, None] + m - n)
    seen = ahead <= 0
    return seen & (ahead > -window) if window else seen


def softmax(s, seen):
    s = s.masked_fill(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(s - torch.where(torch.isinf(top), 0.0, top)), 0.0)
    return e / e.sum(-1, keepdim=True).clamp(min=1e-300)


def ragged(q, k, v, q_at, k_at, window, scale, do=None):
    """``(o, its bound)``, with ``do`` also ``(dq, bound), (dk, bound), (dv, bound)``.

    A weight is rounded to 16 bits (u p), the result once more: |do_i| <= u (sum p |v| + |o|). delta = do . o sees the rounded o, so it is
    off by E = sum_d |do| u (sum p |v| + |o|); dS = p (dP - delta) is rounded: u |dS| + p E; dP - delta adds SMALL of its terms."""
    u = U[q.dtype]
    group, dev = q.size(1) // k.size(1), q.device
    z = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=dev)  # noqa: E731
    o, eo, dq, eq, dk, ek, dv, ev = z(q), z(q), z(q), z(q), z(k), z(k), z(v), z(v)
    for b in range(len(q_at) - 1):
        qs, ks = slice(q_at[b], q_at[b + 1]), slice(k_at[b], k_at[b + 1])
        if qs.stop == qs.start or ks.stop == ks.start:
            continue
        seen = visible(qs.stop - qs.start, ks.stop - ks.start, window, dev)
        for h in range(q.size(1)):
            g = h // group
            qh, kh, vh = q[qs, h].double(), k[ks, g].double(), v[ks, g].double()
            p = softmax(qh @ kh.T * scale, seen)
            o[qs, h] = p @ vh
            eo[qs, h] = (u + SMALL) * (p @ vh.abs()) + u * o[qs, h].abs()
            if do is None:
                continue
            dh = do[qs, h].double()
            dp = dh @ vh.T
            delta = (dh * o[qs, h]).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            off = (dh.abs() * eo[qs, h]).sum(-1, keepdim=True)
            es = (u + SMALL) * ds.abs() + p * (off + SMALL * (dh.abs() @ vh.abs().T + (dh * o[qs, h]).abs().sum(-1, keepdim=True)))
            dq[qs, h] = ds @ kh * scale
            eq[qs, h] = es @ kh.abs() * scale
            dk[ks, g] += ds.T @ qh * scale
            ek[ks, g] += es.T @ qh.abs() * scale
            dv[ks, g] += p.T @ dh
            ev[ks, g] += (u + SMALL) * (p.T @ dh.abs())
    if do is None:
        return o, eo
    return (o, eo), (dq, eq + u * dq.abs()), (dk, ek + u * dk.abs()), (dv, ev + u * dv.abs())


def near(got, want, bound):
    assert got.shape == want.shape
    got = got.double()
    assert torch.isfinite(got).all()
    over = (got - want).abs() - bound - 2.0 ** -24          # a 16-bit result near zero: the type's smallest steps
    assert over.max().item() <= 0 if over.numel() else True, (over.max().item(), (got - want).abs().max().item())


def pages_of(table, b, n, page):
    at = torch.arange(n, device=table.device)
    return table[b].long()[at // page], at % page


def held(pool, scale, table, b, n):
    """The first ``n`` vectors of sequence ``b``: ``[n, heads, D]``."""
    pages, place = pages_of(table, b, n, pool.size(2))
    if scale is None:
        return pool[pages, :, place].double()
    return pool.view(torch.uint8)[pages, :, place].view(torch.float8_e4m3fn).double() * scale[pages, :, place].double()[..., None]


def decode(q, kp, vp, table, lengths, window, scale, ks=None, vs=None):
    """One query per sequence: the result and its bound. With 8-bit pools weights are rounded to f16 relative to the largest value scale
    (2^-11 and less), with 16-bit ones to their type."""
    u, ur = U[q.dtype], U[q.dtype] if ks is None else 2.0 ** -11
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    e = torch.zeros_like(o)
    group = q.size(1) // kp.size(1)
    for b, n in enumerate(lengths):
        first = max(0, n - window) if window else 0
        if n == 0:
            continue
        k, v = (held(p, s, table, b, n)[first:] for p, s in ((kp, ks), (vp, vs)))
        for h in range(q.size(1)):
            p = torch.softmax(k[:, h // group] @ q[b, h].double() * scale, 0)
            o[b, h] = p @ v[:, h // group]
            e[b, h] = (ur + SMALL) * (p @ v[:, h // group].abs()) + u * o[b, h].abs()
            if ks is not None:      # f16 weights below its smallest steps, relative to the largest scale
                e[b, h] += 2.0 ** -25 * n * v[:, h // group].abs().amax(0)
    return o, e


def sample(logits, uniform, temperature, top_k, top_p, min_p):
    """Row by row on lists in Python's own numbers."""
    import math
    out = []
    for r in range(logits.size(0)):
        x, u = logits[r].double().tolist(), float(uniform[r])
        t, k, p, low = (float(s[r]) if torch.is_tensor(s) else s for s in (temperature, top_k, top_p, min_p))
        if any(v != v for v in x) or max(x) == -math.inf or not 0 <= u < 1:
            out.append(-1)
            continue
        top = max(x)
        order = sorted(range(len(x)), key=lambda i: (-x[i], i))
        if not t > 0:
            out.append(order[0])
            continue
        w = {i: 1.0 if x[i] == top else math.exp((x[i] - top) / t) for i in order}
        if k > 0:
            order = order[:int(k)]
        total, ahead, kept = math.fsum(w[i] for i in order), 0.0, []
        for rank, i in enumerate(order):
            if rank and ((p < 1 and ahead > p * total) or w[i] < min(low, 1.0)):
                break
            kept.append(i)
            ahead += w[i]
        goal, total, choice = u * math.fsum(w[i] for i in kept), 0.0, None
        for i in sorted(kept):
            total += w[i]
            if total > goal:
                choice = i
                break
        out.append(choice)
    return torch.tensor(out, device=logits.device)
