"""Oracle: operators on packed sequences, in float64 on the CPU, with what their error bounds need.

TEST INFRASTRUCTURE ONLY - see oracle/__init__.py.

Restates rotary positions and attention over packed sequences from their formulas; the attention also returns, per row
and entry, the sums of magnitudes that a rounding error of a score or a weight is multiplied by.
"""
import math

import torch


def rotary(x, positions, frequencies, layout, offset, amplitude, inverse=False):
    """x [T, H, D] -> (float64 result, sum of the magnitudes of the two products behind each entry)."""
    x = x.double()
    T, H, D = x.shape
    freq = frequencies.reshape(-1).double()
    pairs = freq.numel()
    axes = positions.shape[0] if positions.dim() == 2 else 1
    pos = positions.reshape(axes, T).double()
    out, size = x.clone(), x.abs().clone()
    for i in range(pairs):
        a, b = (offset + i, offset + i + pairs) if layout == "half" else (offset + 2 * i, offset + 2 * i + 1)
        theta = pos[i // (pairs // axes)] * freq[i] * (-1.0 if inverse else 1.0)
        c, s = (theta.cos() * amplitude)[:, None], (theta.sin() * amplitude)[:, None]
        out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        size[..., a] = size[..., b] = abs(amplitude) * (x[..., a].abs() + x[..., b].abs())
    return out, size


def frequencies(part, base, axes, factor, original, low=1.0, high=32.0):
    out = []
    pairs = part // 2 // axes
    for _ in range(axes):
        for i in range(pairs):
            f = base ** (-i / pairs)
            if factor != 1.0:
                turns = 0.0 if original is None else original * f / (2 * math.pi)
                keep = min(1.0, max(0.0, (turns - low) / (high - low))) if original is not None else 0.0
                f = keep * f + (1 - keep) * f / factor
            out.append(f)
    return torch.tensor(out, dtype=torch.float64).reshape(axes, pairs)


def visible(n, m, causal):
    """Boolean [n, m]: which keys the queries of a sequence see."""
    i, j = torch.arange(n)[:, None], torch.arange(m)[None, :]
    return (j <= i + (m - n)) if causal else torch.ones(n, m, dtype=torch.bool)


def attention(q, k, v, starts_q, starts_k, causal, scale=None):
    """-> dict: out [T, H, D], sums [T, H] (float64; zero and -inf where a row sees no key or lies outside), weighted =
    sum_j p_j |v_j|, plain = sum_j |v_j| over the keys seen, score = max_j scale sum_d |q_d k_d|, keys = keys seen."""
    q, k, v = q.double(), k.double(), v.double()
    T, H, D = q.shape
    group = H // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    r = {"out": torch.zeros(T, H, D, dtype=torch.float64), "sums": torch.full((T, H), -math.inf, dtype=torch.float64),
         "weighted": torch.zeros(T, H, D, dtype=torch.float64), "plain": torch.zeros(T, H, D, dtype=torch.float64),
         "score": torch.zeros(T, H, dtype=torch.float64), "keys": torch.zeros(T, H, dtype=torch.float64)}
    sq, sk = [int(x) for x in starts_q], [int(x) for x in starts_k]
    for s in range(len(sq) - 1):
        n, m = sq[s + 1] - sq[s], sk[s + 1] - sk[s]
        if n == 0 or m == 0:
            continue
        seen = visible(n, m, causal)
        some = seen.any(1)
        for h in range(H):
            Q, K, V = q[sq[s]:sq[s + 1], h], k[sk[s]:sk[s + 1], h // group], v[sk[s]:sk[s + 1], h // group]
            x = (Q @ K.T) * scale
            x = torch.where(seen, x, torch.full_like(x, -math.inf))
            top = x.amax(1, keepdim=True)
            top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
            p = torch.exp(x - top)
            total = p.sum(1, keepdim=True)
            p = torch.where(some[:, None], p / torch.where(total > 0, total, torch.ones_like(total)), torch.zeros_like(p))
            V0 = torch.where(seen[:, :, None].any(0).any(0)[None] & torch.isfinite(V), V, torch.zeros_like(V))
            rows = slice(sq[s], sq[s + 1])
            o = p @ V0
            odd = ~torch.isfinite(V)
            if odd.any():                              # what is not finite reaches the rows that see it, and those alone
                for j in odd.any(1).nonzero().flatten().tolist():
                    term = torch.where(odd[j], V[j], torch.zeros_like(V[j]))[None, :] * p[:, j, None]
                    o = torch.where(seen[:, j, None] & odd[j][None, :], o + term, o)
            r["out"][rows, h] = o
            r["sums"][rows, h] = torch.where(some, (top + total.log())[:, 0], torch.full_like(top[:, 0], -math.inf))
            r["weighted"][rows, h] = p @ V0.abs()
            r["plain"][rows, h] = seen.double() @ V0.abs()
            r["score"][rows, h] = torch.where(seen, (Q.abs() @ K.abs().T) * abs(scale), torch.zeros(n, m, dtype=torch.float64)).amax(1)
            r["keys"][rows, h] = seen.double().sum(1)
    return r
