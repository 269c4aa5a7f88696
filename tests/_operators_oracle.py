"""Plain 64-bit implementations of the operators around the expert FFN, written
from their definitions (loops over rows where that is clearest)."""
import numpy as np

NEG = -np.inf


def route_topk(logits, topk, score="softmax", bias=None, num_groups=1, top_groups=None,
               group_best=1, renormalize=True, scale=1.0):
    """(idx int32 [T, K], weights float64 [T, K]) of float64 logits [T, E]."""
    T, E = logits.shape
    per = E // num_groups
    top_groups = num_groups if top_groups is None else top_groups
    idx = np.full((T, topk), -1, np.int32)
    weights = np.zeros((T, topk))
    for t in range(T):
        x = logits[t]
        with np.errstate(all="ignore"):
            if score == "sigmoid":
                s = 1.0 / (1.0 + np.exp(-x))
            else:
                m = np.max(x) if not np.isnan(x).any() else np.nan
                e = np.exp(x - m) if m != NEG else np.zeros(E)
                s = e / e.sum() if m != NEG else e
        c = x.copy() if bias is None else np.where(x == NEG, NEG, s + bias)
        live = c != NEG
        key = lambda v: (1, 0.0) if np.isnan(v) else (0, v)  # noqa: E731  NaN first
        if num_groups > 1:
            worth = []
            for g in range(num_groups):
                own = [e for e in range(g * per, (g + 1) * per) if live[e]]
                own.sort(key=lambda e: key(c[e]), reverse=True)
                if not own:
                    continue
                if group_best == 1:
                    w = c[own[0]]
                else:
                    w = sum((c[e] if bias is not None else s[e]) for e in own[:2])
                worth.append((g, w))
            worth.sort(key=lambda gw: key(gw[1]), reverse=True)  # stable: lowest group first
            kept = {g for g, _ in worth[:top_groups]}
            live = live & np.array([e // per in kept for e in range(E)])
        order = sorted((e for e in range(E) if live[e]), key=lambda e: key(c[e]), reverse=True)
        order = order[:topk]
        if not order:
            continue
        idx[t, :len(order)] = order
        if renormalize and score == "softmax":
            z = x[order]
            with np.errstate(all="ignore"):
                p = np.exp(z - (np.max(z) if not np.isnan(z).any() else np.nan))
            w = p / p.sum()
        else:
            w = s[order]
            if renormalize:
                w = w / w.sum() if w.sum() != 0 else w
        weights[t, :len(order)] = scale * w
    return idx, weights


def route_grad(logits, idx, dw, score="softmax", renormalize=True, scale=1.0):
    """d logits of the weights, the choice held fixed: J^T dw from the full
    Jacobian of every token."""
    T, E = logits.shape
    out = np.zeros((T, E))
    for t in range(T):
        sel = [int(e) for e in idx[t] if e >= 0]
        if not sel:
            continue
        x = logits[t]
        if score == "sigmoid":
            s = 1.0 / (1.0 + np.exp(-x))
            js = np.diag(s * (1.0 / (1.0 + np.exp(x))))
        else:
            e = np.exp(x - x.max())
            s = e / e.sum()
            js = np.diag(s) - np.outer(s, s)
        v, j = s[sel], js[sel]
        if renormalize:
            total = v.sum()
            j = j / total - np.outer(v, j.sum(axis=0)) / total ** 2
        out[t] = scale * (dw[t, :len(sel)] @ j)
    return out


def norm(x, weight=None, bias=None, eps=1e-5, center=True):
    """(y, xhat, r) over the last axis."""
    mu = x.mean(axis=-1, keepdims=True) if center else 0.0
    r = 1.0 / np.sqrt(((x - mu) ** 2).mean(axis=-1, keepdims=True) + eps)
    xhat = (x - mu) * r
    y = xhat * (1.0 if weight is None else weight)
    return (y if bias is None else y + bias), xhat, r


def norm_grad(dy, x, weight=None, eps=1e-5, center=True):
    """(dx, dweight, dbias): dx from the Jacobian of xhat, row by row."""
    _, xhat, r = norm(x, eps=eps, center=center)
    n = x.shape[-1]
    u = dy * (1.0 if weight is None else weight)
    dx = np.zeros_like(x)
    for i in range(x.shape[0]):
        h = xhat[i]
        # d xhat_a / d x_b = r (delta_ab - [1/n] - h_a h_b / n)
        dx[i] = r[i] * (u[i] - (u[i].mean() if center else 0.0) - h * (u[i] @ h) / n)
    return dx, (dy * xhat).sum(axis=0), dy.sum(axis=0)


def adamw(p, g, m, v, step, lr, betas, eps, weight_decay):
    """(p, m, v) after one step, v the second moment itself."""
    b1, b2 = betas
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p * (1 - lr * weight_decay)
    return p - lr * (m / (1 - b1 ** step)) / (np.sqrt(v / (1 - b2 ** step)) + eps), m, v


def mx8_values(q, s):
    """float64 values of an 8-bit state: e4m3 payload bytes, E8M0 scale bytes."""
    q = np.asarray(q, np.uint8).reshape(-1)
    sign = np.where(q & 0x80, -1.0, 1.0)
    e, f = ((q >> 3) & 15).astype(int), (q & 7).astype(float)
    val = np.where(e == 0, f * 2.0 ** -9, (1 + f / 8) * 2.0 ** (e - 7))
    val = np.where((q & 0x7F) == 0x7F, np.nan, val)
    up = np.repeat(2.0 ** (np.asarray(s, np.uint8).reshape(-1).astype(int) - 127), 32)[:q.size]
    return sign * val * up


def linear_cross_entropy(x, w, target, ignore=-100):
    """(token losses, d token loss / d z [T, V]) in float64; ignored tokens 0."""
    z = x @ w.T
    m = z.max(axis=1, keepdims=True)
    p = np.exp(z - m)
    total = p.sum(axis=1, keepdims=True)
    live = target != ignore
    loss = np.zeros(len(target))
    rows = np.arange(len(target))[live]
    loss[live] = (np.log(total) + m)[live, 0] - z[rows, target[live]]
    d = p / total
    d[rows, target[live]] -= 1
    d[~live] = 0
    return loss, d
