"""Plain, slow oracles of the ops of sequences with a common beginning, in float64 and one sequence (or group) at a time. Nothing here is
imported from the package under test."""
import math

import torch


def unit(x, w, eps):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w


def shared_attention(proj, wq, wk, k, v, pos, count, lead, shared, T, H, window, keep, scale, sink, eps, dtype):
    """`proj (B, T, columns)`, caches `k (B, G, S, d)`, `v` in float64, changed in place. New keys are rounded to `dtype`.
    Returns `{(sequence, row): (heads * vdim)}` of the real rows."""
    B, G, S, d = k.shape
    dv, R, out = v.shape[-1], H // G, {}
    before = [x.clone() for x in (k, v)]
    places = {b: (pos[b], min(count[b], T)) for b in range(B) if count[b] > 0 and 0 <= pos[b] <= S - min(count[b], T)}
    for b, (p, n) in places.items():
        for t in range(n):
            row = proj[b, t]
            k[b, :, p + t] = unit(row[H * d:(H + G) * d].reshape(G, d), wk, eps).to(dtype).double()
            v[b, :, p + t] = row[(H + G) * d:(H + G) * d + G * dv].reshape(G, dv)
    for b, (p, n) in places.items():
        edge = max(0, min(shared[b], p, pos[lead[b]])) if 0 <= lead[b] < B else 0
        for t in range(n):
            i, row, heads = p + t, proj[b, t], []
            q = unit(row[:H * d].reshape(H, d), wq, eps)
            seen = torch.tensor([j for j in range(i + 1) if not window or i - j < window or j < keep])
            theirs, own = seen[seen < edge], seen[seen >= edge]
            for h in range(H):
                keys, vals = (torch.cat((old[lead[b], h // R, theirs] if edge else old[b, h // R, :0], x[b, h // R, own])) for old, x in zip(before, (k, v)))
                s = keys @ q[h] * scale
                if sink is not None:
                    s = torch.cat((s, torch.tensor([float(sink)], dtype=torch.float64)))
                heads.append(torch.softmax(s, 0)[:len(seen)] @ vals)
            o = torch.cat(heads)
            if len(row) > (H + G) * d + G * dv:
                o = o * torch.sigmoid(row[(H + G) * d + G * dv:])
            out[b, t] = o
    return out


def next_beams(logits, scores, ended, length, K, end, valid, penalty):
    """The next beams of one group: `[(slot, parent, token, sum, ended, length)]` by slots within the group; None: it has none."""
    scores = [float(s) if math.isfinite(s) else -math.inf for s in scores]
    if all(s == -math.inf for s in scores):
        return None
    found = []
    for k in range(K):
        done = end is not None and bool(ended[k])
        after = int(length[k]) + (not done)
        if done:
            c = torch.full((valid,), -math.inf, dtype=torch.float64)
            c[end] = scores[k]
        else:
            x = logits[k, :valid].double()
            x[torch.isnan(x)] = -math.inf
            c = scores[k] + torch.log_softmax(x, 0)
            c[torch.isnan(c)] = -math.inf
        best = torch.sort(c, descending=True, stable=True)
        found += [(-float(y) / max(after, 1) ** penalty, k, int(i), float(y), done, after) for y, i in zip(best.values[:K], best.indices[:K])]
    found = sorted(found, key=lambda f: f[:3])[:K]
    free, taken, out = [s for s in range(K) if s not in {f[1] for f in found}], set(), []
    for _, k, token, c, done, after in found:
        slot = free.pop(0) if k in taken else k
        taken.add(k)
        out.append((slot, k, token, c, int(done or token == end), after))
    return sorted(out)


def reordered(x, parent, begin, end, K, axis, per):
    """A state after its rows have followed their parents."""
    out = x.clone()
    for b, p in enumerate(parent):
        if p // K != b // K or not 0 <= p < x.shape[0]:
            continue
        if axis is None:
            out[b] = x[p]
            continue
        for i in range(x.shape[axis]):
            if any(begin[b] <= j < end[b] for j in range(i * per, (i + 1) * per)):
                out[b].select(axis - 1, i).copy_(x[p].select(axis - 1, i))
    return out
