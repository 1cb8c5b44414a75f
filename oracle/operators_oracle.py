"""Plain 64-bit CPU forms of the operators on grouped rows and of the gated scan (nerf_amd.ops), written from their
formulas, with for every output a magnitude: the same sum with absolute values, which is what rounding errors scale with.

The reference has no counterpart of these operators: parity unpinned."""
import torch


def cpu64(t):
    return None if t is None else t.detach().cpu().double()


def group_rows(ids, n_groups):
    """(order, offsets) by counting"""
    buckets = [[] for _ in range(n_groups + 1)]
    for i, v in enumerate(ids.detach().cpu().tolist()):
        buckets[v if 0 <= v < n_groups else n_groups].append(i)
    offsets = [0]
    for b in buckets[:n_groups]:
        offsets.append(offsets[-1] + len(b))
    return (torch.tensor([i for b in buckets for i in b], dtype=torch.int64).reshape(-1), torch.tensor(offsets, dtype=torch.int64))


def embed_rows(ids, table, scale):
    """(out, |out|)"""
    ids, table = ids.detach().cpu().reshape(-1), cpu64(table)
    ok = (ids >= 0) & (ids < table.shape[0])
    out = torch.zeros((ids.numel(), table.shape[1]), dtype=torch.float64)
    out[ok] = table[ids[ok]] * scale
    return out, out.abs()


def embed_rows_grad(ids, rows, d_out, scale):
    """(d_table, magnitude, rows summed)"""
    ids, g = ids.detach().cpu().reshape(-1).long(), cpu64(d_out)
    g = g.reshape(ids.numel(), -1)
    ok = (ids >= 0) & (ids < rows)
    d, m = (torch.zeros((rows, g.shape[1]), dtype=torch.float64) for _ in range(2))
    d.index_add_(0, ids[ok], g[ok] * scale)
    m.index_add_(0, ids[ok], (g[ok] * scale).abs())
    return d, m, torch.bincount(ids[ok], minlength=rows)


def grouped_linear(x, weight, bias, rows_of, relu):
    """rows_of[g]: the rows of group g.  (z before the ReLU cut, y, magnitude)"""
    x, w, b = cpu64(x), cpu64(weight), cpu64(bias)
    G, N, K = w.shape
    y, m = (torch.zeros((x.shape[0], N), dtype=torch.float64) for _ in range(2))
    for g in range(G):
        r = rows_of[g]
        y[r] = x[r] @ w[g].T + (b[g] if b is not None else 0.0)
        m[r] = x[r].abs() @ w[g].abs().T + (b[g].abs() if b is not None else 0.0)
    return (torch.where(y < 0, torch.zeros_like(y), y) if relu else y), m


def grouped_linear_grads(x, weight, rows_of, d_y, y=None):
    """d_x, d_weight, d_bias, each with its magnitude; y: the layer's output where it had a ReLU"""
    x, w, g_out = cpu64(x), cpu64(weight), cpu64(d_y)
    if y is not None:
        g_out = torch.where(cpu64(y) <= 0, torch.zeros_like(g_out), g_out)
    dx, mx = torch.zeros_like(x), torch.zeros_like(x)
    dw, mw = torch.zeros_like(w), torch.zeros_like(w)
    db, mb = (torch.zeros(w.shape[:2], dtype=torch.float64) for _ in range(2))
    for g in range(w.shape[0]):
        r = rows_of[g]
        dx[r], mx[r] = g_out[r] @ w[g], g_out[r].abs() @ w[g].abs()
        dw[g], mw[g] = g_out[r].T @ x[r], g_out[r].abs().T @ x[r].abs()
        db[g], mb[g] = g_out[r].sum(0), g_out[r].abs().sum(0)
    return (dx, mx), (dw, mw), (db, mb)


def gated_scan(gate, value, state, reverse):
    """(h, |h|, last, |last|) step by step"""
    a, v = cpu64(gate), cpu64(value)
    B, T, D = v.shape
    a = a.expand(B, T, a.shape[2])
    h = torch.zeros((B, D), dtype=torch.float64) if state is None else cpu64(state)
    m = h.abs()
    out, mag = torch.zeros_like(v), torch.zeros_like(v)
    for t in (range(T - 1, -1, -1) if reverse else range(T)):
        h = a[:, t] * h + v[:, t]
        m = a[:, t].abs() * m + v[:, t].abs()
        out[:, t], mag[:, t] = h, m
    return out, mag, h, m


def gated_scan_grads(gate, value, state, reverse, d_h, d_last):
    """d_gate (of the gate's own last size), d_value, d_state, each with its magnitude"""
    a, v = cpu64(gate), cpu64(value)
    B, T, D = v.shape
    shared = a.shape[2] == 1 and D > 1
    a = a.expand(B, T, a.shape[2])
    h0 = torch.zeros((B, D), dtype=torch.float64) if state is None else cpu64(state)
    out, mag, _, _ = gated_scan(gate, value, state, reverse)
    steps = list(range(T - 1, -1, -1) if reverse else range(T))
    u = torch.zeros((B, D), dtype=torch.float64) if d_last is None else cpu64(d_last)
    mu = u.abs()
    g_out = torch.zeros_like(v) if d_h is None else cpu64(d_h)
    dv, mv, da, ma = (torch.zeros_like(v) for _ in range(4))
    for i in range(T - 1, -1, -1):
        t = steps[i]
        G, mG = g_out[:, t] + u, g_out[:, t].abs() + mu
        before, mbefore = (h0, h0.abs()) if i == 0 else (out[:, steps[i - 1]], mag[:, steps[i - 1]])
        dv[:, t], mv[:, t] = G, mG
        da[:, t], ma[:, t] = G * before, mG * mbefore
        u, mu = a[:, t] * G, a[:, t].abs() * mG
    if shared:
        da, ma = da.sum(2, keepdim=True), ma.sum(2, keepdim=True)
    return (da, ma), (dv, mv), (u, mu)
