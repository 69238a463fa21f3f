"""Oracle for the operators of ragged batches, in 64 bits from the formulas, with how far a kernel may be off.

The bounds count roundings.  With A = sum_j p_j |v_j| (the weights are positive and sum to 1) an output is off by at most
  u |o|        its own rounding, u = eps / 2 of the 16-bit type,
  u A          the weights' rounding to that type (weights below the normal range: half a subnormal step each),
  2 d A        the scores' error d, in numerator and denominator: a product of D terms in fp32, each term and each sum off by 2^-23 of
               sum |q_i k_i| at most (tensor cores may drop the last bit instead of rounding it), and the exponential's 2^-21,
  n 2^-23 A    the sum over n keys in fp32, and as much for the denominator.
"""
import math

import torch


def attend(q, k, v, limit, scale, kind):
    """q [n, H, D], k and v [m, G, D] (any float type); query i sees the keys j < limit[i].  -> (o, bound) in float64."""
    n, H, D = q.shape
    m, G = k.shape[0], k.shape[1]
    out, bound = torch.zeros(n, H, D, dtype=torch.float64, device=q.device), torch.zeros(n, H, D, dtype=torch.float64, device=q.device)
    if n == 0 or m == 0:
        return out, bound
    u = torch.finfo(kind).eps / 2
    see = torch.arange(m, device=q.device) < limit[:, None]
    for h in range(H):
        g = h * G // H
        a, b, c = q[:, h].double(), k[:, g].double(), v[:, g].double()
        # what a query does not see takes part in nothing: per-row copies where values may be no numbers
        s = (a @ b.T * scale).masked_fill(~see, -math.inf)
        some = see.any(1)
        e = torch.where(some[:, None], torch.softmax(torch.where(some[:, None], s, 0.0), 1), 0.0)
        e = e.masked_fill(~see, 0.0)
        if torch.isfinite(c).all():
            o, A, vmax = e @ c, e @ c.abs(), c.abs().max()
        else:
            c3 = torch.where(see[:, :, None], c[None], 0.0)
            o, A, vmax = (e[:, :, None] * c3).sum(1), (e[:, :, None] * c3.abs()).sum(1), torch.where(torch.isfinite(c), c.abs(), 0.0).max()
        mags = torch.nan_to_num(a).abs() @ torch.nan_to_num(b).abs().T * scale
        d = (D + 4) * 2.0 ** -23 * mags.masked_fill(~see, 0.0).amax(1, keepdim=True) + 2.0 ** -21
        tiny = m * 2.0 ** -25 * vmax if kind == torch.float16 else 0.0
        out[:, h] = o
        bound[:, h] = u * o.abs() + (u + 2 * d + 2 * m * 2.0 ** -23) * A + tiny + torch.finfo(kind).tiny
    return out, bound


def packed(Q, K, V, q_at, k_at, causal, scale=None):
    """q_at, k_at: lists of batch + 1 offsets.  Rows outside all sequences are NaN in the first result."""
    scale = Q.shape[2] ** -0.5 if scale is None else scale
    out = torch.full(Q.shape, math.nan, dtype=torch.float64, device=Q.device)
    bound = torch.zeros(Q.shape, dtype=torch.float64, device=Q.device)
    for b in range(len(q_at) - 1):
        n, m = q_at[b + 1] - q_at[b], k_at[b + 1] - k_at[b]
        limit = torch.arange(n, device=Q.device) + (m - n + 1) if causal else torch.full((n,), m, device=Q.device)
        rows, keys = slice(q_at[b], q_at[b + 1]), slice(k_at[b], k_at[b + 1])
        out[rows], bound[rows] = attend(Q[rows], K[keys], V[keys], limit.clamp(max=m), scale, Q.dtype)
    return out, bound


def shared(q, K_prefix, V_prefix, K, V, lengths, prefix_len, scale=None):
    """lengths: a list.  The caches are head-major: [kv_heads, keys, D] and [batch, kv_heads, keys, D]."""
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, n in enumerate(lengths):
        k, v = (torch.cat([p[:, :prefix_len], own[b, :, :n]], 1).transpose(0, 1) for p, own in ((K_prefix, K), (V_prefix, V)))
        o, t = attend(q[b:b + 1], k, v, torch.tensor([prefix_len + n], device=q.device), scale, q.dtype)
        out[b], bound[b] = o[0], t[0]
    return out, bound


def adjusted(logits, prompt=None, prompt_lengths=None, tokens=None, token_lengths=None, repetition=None, presence=None, frequency=None,
             bias_ids=None, bias_values=None, mask=None, mask_rows=None):
    """The rules on logits, token by token, on the CPU.  -> (values, bound) in float64."""
    kind = logits.dtype
    x = logits.double().cpu()
    R, V = x.shape
    mag = x.abs()                                            # what has been added so far: each operation is off by half a step of it
    lst = lambda t: None if t is None else t.cpu().tolist()
    prompt, prompt_lengths, tokens, token_lengths, bias_ids, mask, mask_rows = map(lst, (prompt, prompt_lengths, tokens, token_lengths, bias_ids, mask, mask_rows))
    num = lambda t, r, other: other if t is None else float(t.double().cpu()[r])
    values = None if bias_values is None else bias_values.double().cpu().tolist()

    def counted(ids, lengths, r):
        if ids is None:
            return []
        n = len(ids[r]) if lengths is None else min(max(lengths[r], 0), len(ids[r]))
        return [t for t in ids[r][:n] if 0 <= t < V]

    for r in range(R):
        said = {}
        for t in counted(tokens, token_lengths, r):
            said[t] = said.get(t, 0) + 1
        for t in set(said) | set(counted(prompt, prompt_lengths, r)):
            rep = num(repetition, r, 1.0)
            x[r, t] = x[r, t] / rep if x[r, t] > 0 else x[r, t] * rep
            mag[r, t] = max(float(mag[r, t]), abs(float(x[r, t])))
        for t, c in said.items():
            f, p = num(frequency, r, 0.0) * c, num(presence, r, 0.0)
            x[r, t] = x[r, t] - f - p
            mag[r, t] += abs(f) + abs(p)
        for i in range(len(bias_ids[r]) if bias_ids is not None else 0):
            t = bias_ids[r][i]
            if 0 <= t < V:
                x[r, t] += values[r][i]
                mag[r, t] += abs(values[r][i])
        if mask is not None:
            which = r if mask_rows is None else mask_rows[r]
            if 0 <= which < len(mask):
                for t in range(V):
                    if not mask[which][t // 32] >> (t % 32) & 1:
                        x[r, t] = -math.inf
    steps = 6 + (0 if bias_ids is None else len(bias_ids[0]))
    bound = steps * 2.0 ** -24 * mag + torch.finfo(kind).eps / 2 * torch.where(torch.isfinite(x), x.abs(), 0.0) + torch.finfo(kind).tiny
    return x, bound
