"""Plain float64 statements of the layer norm and of the routing by scores, row by row and expert by expert (numpy loops, no
torch operators that could share a mistake with the code under test).  Inputs are numpy arrays of the stored values."""
import math

import numpy as np


def layer_norm(h, weight, bias, eps):
    """(out, mean, rstd) of the rows of h."""
    h = h.astype(np.float64)
    mean = h.sum(1) / h.shape[1]
    c = h - mean[:, None]
    rstd = 1.0 / np.sqrt((c * c).sum(1) / h.shape[1] + eps)
    out = c * rstd[:, None]
    if weight is not None:
        out = out * weight.astype(np.float64)
    if bias is not None:
        out = out + bias.astype(np.float64)
    return out, mean, rstd


def layer_norm_grads(g, gs, h, weight, eps):
    """(grad, grad_weight, grad_bias) from the definition's derivative, written as the full Jacobian of each row:
    d n_i / d h_j = r (delta_ij - 1/D - n_i n_j / D)."""
    _, mean, rstd = layer_norm(h, None, None, eps)
    g = g.astype(np.float64)
    n = (h.astype(np.float64) - mean[:, None]) * rstd[:, None]
    u = g if weight is None else g * weight.astype(np.float64)
    D = h.shape[1]
    grad = np.empty_like(n)
    for row in range(h.shape[0]):
        grad[row] = rstd[row] * (u[row] - u[row].sum() / D - n[row] * (n[row] @ u[row]) / D)
    if gs is not None:
        grad = grad + gs.astype(np.float64)
    return grad, (g * n).sum(0), g.sum(0)


def _scores(z, scoring):
    if scoring == 'softmax':
        top = max(z)
        e = [math.exp(v - top) if v > -math.inf else 0.0 for v in z]
        return [v / sum(e) for v in e]
    return [1.0 / (1.0 + math.exp(-v)) if v > -700 else (math.exp(v) if v > -math.inf else 0.0) for v in z]


def route_row(z, k, scoring, bias=None, n_groups=1, kept_groups=1, group_score='top2', renormalise=True, scale=1.0):
    """(indices, weights) of one row of logits, places left over as (-1, 0)."""
    z = [float(v) for v in z]
    E = len(z)
    nothing = [-1] * k, [0.0] * k
    if any(math.isnan(v) or (scoring == 'softmax' and v == math.inf) for v in z) or all(v == -math.inf for v in z):
        return nothing
    s = _scores(z, scoring)
    if bias is None and not (n_groups > 1 and group_score == 'top2'):
        c = list(z)
    else:
        c = [a + (0.0 if bias is None else float(bias[e])) for e, a in enumerate(s)]
    if any(math.isnan(v) for v in c):
        return nothing
    c = [-math.inf if v == -math.inf else w for v, w in zip(z, c)]
    size = E // n_groups
    open_groups = list(range(n_groups))
    if n_groups > 1:
        def score(i):
            best = sorted(c[i * size:(i + 1) * size], reverse=True)
            return best[0] + best[1] if group_score == 'top2' and size > 1 and best[1] > -math.inf else best[0]
        open_groups = sorted(range(n_groups), key=lambda i: (-score(i), i))[:kept_groups]
    order = sorted((e for e in range(E) if e // size in open_groups and c[e] > -math.inf), key=lambda e: (-c[e], e))[:k]
    if scoring == 'softmax':
        top = max(z[e] for e in order) if order else 0.0
        part = {e: math.exp(z[e] - top) for e in order}          # s up to a common factor, free of underflow
    else:
        top = max(min(z[e], 0.0) for e in order) if order else 0.0
        part = {e: math.exp(min(z[e], 0.0) - top) / (1.0 + math.exp(-abs(z[e]))) for e in order}
    w = {e: scale * (part[e] / sum(part.values()) if renormalise else s[e]) for e in order}
    left = k - len(order)
    return order + [-1] * left, [w[e] for e in order] + [0.0] * left


def route(z, k, scoring, **kw):
    rows = [route_row(r, k, scoring, **kw) for r in z]
    idx = np.array([r[0] for r in rows], dtype=np.int64).reshape(len(z), k)
    w = np.array([r[1] for r in rows], dtype=np.float64).reshape(len(z), k)
    dense = np.zeros(z.shape, dtype=np.float64)
    for n in range(len(z)):
        for i in range(k):
            if idx[n, i] >= 0:
                dense[n, idx[n, i]] = w[n, i]
    return dense, idx, w


def route_grads(z, idx, q, scoring, renormalise, scale):
    """Gradient of the logits from the gradient q of the weights by place, as the product with the Jacobian of each row."""
    out = np.zeros(z.shape, dtype=np.float64)
    for n in range(z.shape[0]):
        chosen = [(i, e) for i, e in enumerate(idx[n]) if 0 <= e < z.shape[1]]
        if not chosen:
            continue
        s = _scores([float(v) for v in z[n]], scoring)
        if renormalise:
            row_z = [float(z[n, e]) for _, e in chosen]
            if scoring == 'softmax':
                part = [math.exp(v - max(row_z)) for v in row_z]
            else:
                low = max(min(v, 0.0) for v in row_z)
                part = [math.exp(min(v, 0.0) - low) / (1.0 + math.exp(-abs(v))) for v in row_z]
            p = [v / sum(part) for v in part]
            for a, (_, e) in enumerate(chosen):
                d = sum(q[n, i] * scale * p[b] * ((1.0 if a == b else 0.0) - p[a]) for b, (i, _) in enumerate(chosen))
                if scoring == 'sigmoid':
                    d *= 1.0 / (1.0 + math.exp(z[n, e])) if z[n, e] < 700 else 0.0
                out[n, e] += d
        else:
            for i, e in chosen:
                if scoring == 'sigmoid':
                    out[n, e] += scale * q[n, i] * s[e] * (1.0 / (1.0 + math.exp(z[n, e])) if z[n, e] < 700 else 0.0)
                else:
                    for j in range(z.shape[1]):
                        out[n, j] += scale * q[n, i] * s[e] * ((1.0 if j == e else 0.0) - s[j])
    return out
