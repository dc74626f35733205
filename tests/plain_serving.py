"""Plain, slow oracle of the serving ops: whole sequences at once, elementary torch expressions in float64. Nothing here is
imported from the package under test."""
import torch

BLOCK = 64


def heads_rms(x, w, eps):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w


def block_codes(block):
    """Codes `(64, width)` and scale of one head's complete block. The scale is a float32 quotient, and codes are the nearest whole
    numbers to float32 quotients: both are part of the definition."""
    top = block.abs().max().float()
    scale = top / torch.tensor(127.0)
    if scale == 0:
        return torch.zeros_like(block), scale
    return torch.round(block.float() / scale).double(), scale


def q8_attention(rows, q_norm, k_norm, heads, G, dim, vdim, window, keep, scale, sink, eps, dtype):
    """One sequence, all its tokens at once: `rows (n, [q | k | v | gate])` float64. Returns `(outputs (n, heads * vdim), keys,
    values)`, keys and values `(n, G, width)` in float64 as `dtype` holds them."""
    n, R = rows.shape[0], heads // G
    q, k, v, gate = rows.split((heads * dim, G * dim, G * vdim, rows.shape[1] - (heads + G) * dim - G * vdim), 1)
    q = heads_rms(q.reshape(n, heads, dim), q_norm, eps)
    k = heads_rms(k.reshape(n, G, dim), k_norm, eps).to(dtype).double()
    v = v.reshape(n, G, vdim)
    kq, vq = k.clone(), v.clone()  # what later blocks see
    for lo in range(0, n // BLOCK * BLOCK, BLOCK):
        for g in range(G):
            for held, x in ((kq, k), (vq, v)):
                codes, step = block_codes(x[lo:lo + BLOCK, g])
                held[lo:lo + BLOCK, g] = codes * step.double()
    out = torch.zeros(n, G, R, vdim, dtype=torch.float64)
    for i in range(n):
        j = torch.arange(i + 1)
        if window:
            j = j[(i - j < window) | (j < keep)]
        own = (j >= i // BLOCK * BLOCK)[:, None, None]
        keys, vals = (torch.where(own, a[j], b[j]).transpose(0, 1) for a, b in ((k, kq), (v, vq)))
        s = q[i].reshape(G, R, dim) @ keys.transpose(1, 2) * scale
        top = s.amax(-1, keepdim=True)
        if sink is not None:
            top = top.clamp(min=sink)
        e = torch.exp(s - top)
        out[i] = (e @ vals) / (e.sum(-1, keepdim=True) + (0.0 if sink is None else torch.exp(sink - top)))
    out = out.reshape(n, heads * vdim)
    return (out * torch.sigmoid(gate) if gate.shape[1] else out), k, v


def adapted(x, w, a, b, scale, slot, T):
    y = x @ w.T
    for i, s in enumerate(slot):
        if 0 <= s < len(a):
            y[i * T:(i + 1) * T] += scale[s] * (x[i * T:(i + 1) * T] @ a[s].T @ b[s].T)
    return y


def shaped(x, history, start, penalties, biases, allowed):
    """One row: `history` its tokens in order, `biases` a list of (token, value), `allowed` a list of truth values."""
    repetition, frequency, presence = (float(p) for p in penalties)
    x = [float(v) for v in x]
    for t in set(history):
        if 0 <= t < len(x):
            x[t] = x[t] / repetition if x[t] > 0 else x[t] * repetition
    later = history[start:]
    for t in set(later):
        if 0 <= t < len(x):
            x[t] = x[t] - frequency * later.count(t) - presence
    for t, v in biases:
        if 0 <= t < len(x):
            x[t] += float(v)
    return torch.tensor([v if ok else float("-inf") for v, ok in zip(x, allowed)], dtype=torch.float64)
