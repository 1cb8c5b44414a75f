"""Cases and plain forms of the index-conditional operators and the scan along rays.

Four operators that belong together in a radiance field whose sub-networks are chosen by an id:

``group_rows``      ids [n] -> the stable order that puts the rows of one group next to each other, and where each
                    group begins (the router's hand-over to the experts' products).
``embed_rows``      out[i] = scale * table[ids[i]] and the table's gradient (per-image codes, feature tables).
``grouped_linear``  y[i] = W[g(i)] x[i] + b[g(i)] for rows of ragged groups, with its three gradients.
``gated_scan``      h[t] = a[t] h[t-1] + v[t] along the samples of a ray, front to back or back to front, with its
                    gradients (a is one gate per sample, as 1 - alpha in compositing, or one per channel).

An id outside [0, n_groups) belongs to no group: its rows come last in the order and give zeros.

``run`` computes the plain form with elementary torch operations in 32 bits while ``own`` is False, and calls
nerf_amd where it is True.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ----------------------------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # the router of one training batch: 1024 rays over 8 sub-networks; a call is all latency
        {"name": "group batch", "op": "group", "n": 1024, "groups": 8, "ids": "uniform"},
        # every sample point of 4096 rays x 192 samples over a grid of 64 sub-networks
        {"name": "group samples", "op": "group", "n": 786432, "groups": 64, "ids": "runs"},
        # the per-image codes of a 1024-ray batch drawn from 100 images, one training pass
        {"name": "codes batch", "op": "embed", "n": 1024, "rows": 100, "dim": 48, "dtype": "fp32", "ids": "uniform", "train": True},
        # the same codes looked up for every sample of the batch: 192 samples of a ray share an id, few rows, long sums
        {"name": "codes samples", "op": "embed", "n": 196608, "rows": 300, "dim": 48, "dtype": "bf16", "ids": "runs", "train": True},
        # a large feature table read at points whose cells repeat unevenly
        {"name": "table", "op": "embed", "n": 524288, "rows": 65536, "dim": 128, "dtype": "fp16", "ids": "skewed", "train": True},
        # first layer of 8 sub-networks on one small chunk: 63 encoded features, rows that are not 16-byte aligned
        {"name": "experts encoded", "op": "linear", "n": 1024, "groups": 8, "k": 63, "m": 256, "dtype": "bf16", "ids": "uniform",
         "relu": True, "train": False},
        # hidden layer 256 -> 256 over all samples of a 1024-ray batch, forward and backward
        {"name": "experts hidden", "op": "linear", "n": 196608, "groups": 8, "k": 256, "m": 256, "dtype": "bf16", "ids": "uniform",
         "relu": False, "train": True},
        # the same layer in the validation precision
        {"name": "experts hidden fp32", "op": "linear", "n": 65536, "groups": 8, "k": 256, "m": 256, "dtype": "fp32",
         "ids": "uniform", "relu": False, "train": True},
        # wide layers, many ragged groups of very different sizes, inference
        {"name": "experts wide", "op": "linear", "n": 65536, "groups": 64, "k": 1024, "m": 1024, "dtype": "fp16", "ids": "skewed",
         "relu": True, "train": False},
        # one step of 1024 marching rays: the state moves on by one sample
        {"name": "scan step", "op": "scan", "b": 1024, "t": 1, "d": 256, "dtype": "fp32", "gate": "shared", "reverse": False,
         "state": True, "train": False},
        # feature compositing back to front over 192 samples of 4096 rays, one gate per sample, forward and backward
        {"name": "scan rays", "op": "scan", "b": 4096, "t": 192, "d": 64, "dtype": "bf16", "gate": "shared", "reverse": True,
         "state": False, "train": True},
        # two very long sequences with a gate per channel, forward and backward
        {"name": "scan long", "op": "scan", "b": 2, "t": 262144, "d": 64, "dtype": "fp32", "gate": "channel", "reverse": False,
         "state": True, "train": True},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["group", "embed", "linear", "linear", "scan", "scan"])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    ids = rng.choice(["uniform", "runs", "skewed"])
    train = rng.random() < 0.6
    if op == "group":
        return {"op": op, "n": _log(rng, 1, 786432), "groups": _log(rng, 1, 4096), "ids": ids}
    if op == "embed":
        dim = _log(rng, 1, 1024)
        return {"op": op, "n": _log(rng, 1, min(524288, (1 << 26) // dim)), "rows": _log(rng, 1, min(131072, (1 << 24) // dim)), "dim": dim,
                "dtype": dtype, "ids": ids, "train": train}
    if op == "linear":
        k, m = _log(rng, 1, 1024), _log(rng, 1, 1024)
        macs = 1 << (31 if dtype == "fp32" else 33)
        return {"op": op, "n": _log(rng, 1, max(1, min(196608, macs // (k * m)))), "groups": _log(rng, 1, 96), "k": k, "m": m,
                "dtype": dtype, "ids": ids, "relu": (not train) and rng.random() < 0.5, "train": train}
    d = _log(rng, 1, 1024)
    t = _log(rng, 1, min(262144, (1 << 24) // d))
    return {"op": op, "b": _log(rng, 1, max(1, min(8192, (1 << 24) // (d * t)))), "t": t, "d": d, "dtype": dtype,
            "gate": rng.choice(["shared", "channel"]), "reverse": rng.random() < 0.5, "state": rng.random() < 0.5, "train": train}


# ----------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------

def _ids(gen, n, groups, kind):
    """Group ids: spread evenly, in runs of neighbouring rows (samples of a ray), or a few groups holding most rows.
    About one row in fifty belongs to no group."""
    if kind == "runs":
        per = 192
        ids = torch.randint(0, groups, ((n + per - 1) // per,), generator=gen, device=DEV).repeat_interleave(per)[:n]
    elif kind == "skewed":
        u = torch.rand((n,), generator=gen, device=DEV, dtype=torch.float64)
        ids = (groups * u ** 3).long().clamp_(max=groups - 1)
    else:
        ids = torch.randint(0, groups, (n,), generator=gen, device=DEV)
    none = torch.rand((n,), generator=gen, device=DEV) < 0.02
    return torch.where(none, torch.full_like(ids, -1), ids)


def _order(ids, groups):
    key = torch.where((ids >= 0) & (ids < groups), ids, torch.full_like(ids, groups))
    key, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(key, torch.arange(groups + 1, device=key.device))
    return order.to(torch.int32), offsets.to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape, dtype, scale=1.0):
        return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)

    s = {"case": dict(case)}
    op = case["op"]
    if op == "group":
        s["ids"] = _ids(gen, case["n"], case["groups"], case["ids"])
        return s
    dt = DTYPES[case["dtype"]]
    train = case["train"]
    if op == "embed":
        s["ids"] = _ids(gen, case["n"], case["rows"], case["ids"])
        s["table"] = randn(case["rows"], case["dim"], dtype=dt).requires_grad_(train)
        s["scale"] = math.sqrt(case["dim"])
        if train:
            s["d_out"] = randn(case["n"], case["dim"], dtype=dt)
        return s
    if op == "linear":
        n, g, k, m = case["n"], case["groups"], case["k"], case["m"]
        s["ids"] = _ids(gen, n, g, case["ids"])
        s["x"] = randn(n, k, dtype=dt).requires_grad_(train)
        bound = 1.0 / math.sqrt(k)          # the spread of a fresh linear layer
        s["weight"] = ((torch.rand((g, m, k), generator=gen, device=DEV) * 2 - 1) * bound).to(dt).requires_grad_(train)
        s["bias"] = ((torch.rand((g, m), generator=gen, device=DEV) * 2 - 1) * bound).to(dt).requires_grad_(train)
        if train:
            s["d_out"] = randn(n, m, dtype=dt)
        if own:
            from nerf_amd import ops
            s["groups"] = ops.group_rows(s["ids"], g)        # one routing serves all layers of the sub-networks
        else:
            order, offsets = _order(s["ids"], g)
            s["order"], s["offsets"] = order.long(), offsets.tolist()   # a loop over groups needs their sizes on the host
        return s
    b, t, d = case["b"], case["t"], case["d"]
    # gates as exp(-sigma * delta) gives them: empty space near 1, surfaces near 0
    sigma = torch.rand((b, t, 1 if case["gate"] == "shared" else d), generator=gen, device=DEV)
    s["gate"] = torch.exp(-4.0 * sigma ** 6).to(dt).requires_grad_(train)
    s["value"] = randn(b, t, d, dtype=dt).requires_grad_(train)
    s["state"] = randn(b, d, dtype=torch.float32).requires_grad_(train) if case["state"] else None
    if train:
        s["d_h"] = randn(b, t, d, dtype=dt)
        s["d_last"] = randn(b, d, dtype=torch.float32)
    return s


# ----------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from nerf_amd import ops
    c = s["case"]
    if c["op"] == "group":
        g = ops.group_rows(s["ids"], c["groups"])
        return {"order": g.order, "offsets": g.offsets}
    if c["op"] == "embed":
        out = ops.embed_rows(s["ids"], s["table"], s["scale"])
        if not c["train"]:
            return {"out": out}
        (d_table,) = torch.autograd.grad(out, (s["table"],), s["d_out"])
        return {"out": out.detach(), "d_table": d_table}
    if c["op"] == "linear":
        y = ops.grouped_linear(s["x"], s["weight"], s["groups"], bias=s["bias"], relu=c["relu"])
        if not c["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["d_out"])
        return {"y": y.detach(), "d_x": dx, "d_weight": dw, "d_bias": db}
    h, last = ops.gated_scan(s["gate"], s["value"], state=s["state"], reverse=c["reverse"])
    if not c["train"]:
        return {"h": h, "last": last}
    leaves = [s["gate"], s["value"]] + ([s["state"]] if s["state"] is not None else [])
    grads = torch.autograd.grad((h, last), leaves, (s["d_h"], s["d_last"]))
    return dict(zip(("h", "last", "d_gate", "d_value", "d_state"), (h.detach(), last.detach()) + tuple(grads)))


@torch.no_grad()
def _run_plain(s):
    c = s["case"]
    if c["op"] == "group":
        order, offsets = _order(s["ids"], c["groups"])
        return {"order": order, "offsets": offsets}
    dt = DTYPES[c["dtype"]]
    if c["op"] == "embed":
        ids, table = s["ids"], s["table"]
        ok = (ids >= 0) & (ids < c["rows"])
        at = torch.where(ok, ids, torch.zeros_like(ids))
        out = torch.where(ok[:, None], table[at].float() * s["scale"], 0.0).to(dt)
        if not c["train"]:
            return {"out": out}
        wide = torch.float64 if dt is torch.float32 else torch.float32        # one row may sum half a million terms
        g = torch.where(ok[:, None], s["d_out"].to(wide), 0.0)
        d_table = torch.zeros(table.shape, dtype=wide, device=table.device).index_add_(0, at, g) * s["scale"]
        return {"out": out, "d_table": d_table.to(dt)}
    if c["op"] == "linear":
        return _plain_linear(s, c, dt)
    return _plain_scan(s, c, dt)


def _plain_linear(s, c, dt):
    x, w, b, order, off = s["x"], s["weight"], s["bias"], s["order"], s["offsets"]
    y = torch.zeros((c["n"], c["m"]), dtype=dt, device=x.device)
    if c["train"]:
        dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    for e in range(c["groups"]):
        rows = order[off[e]:off[e + 1]]
        if rows.numel() == 0:
            continue
        xe, we = x[rows].float(), w[e].float()
        z = xe @ we.T + b[e].float()
        y[rows] = (torch.where(z > 0, z, 0.0) if c["relu"] else z).to(dt)
        if c["train"]:
            ge = s["d_out"][rows].float()
            dx[rows] = (ge @ we).to(dt)
            dw[e] = (ge.T @ xe).to(dt)
            db[e] = ge.sum(0).to(dt)
    return {"y": y, "d_x": dx, "d_weight": dw, "d_bias": db} if c["train"] else {"y": y}


def _doubling(a, v):
    """Every prefix of h[t] = a[t] h[t-1] + v[t] from a zero state along dim 1, in log2(T) rounds, and the running
    products of a."""
    a = a.expand_as(v).clone() if a.shape != v.shape else a.clone()
    v = v.clone()
    step, T = 1, v.shape[1]
    while step < T:
        v[:, step:] = v[:, step:] + a[:, step:] * v[:, :-step]
        a[:, step:] = a[:, step:] * a[:, :-step]
        step *= 2
    return a, v


def _plain_scan(s, c, dt):
    a, v = s["gate"].float(), s["value"].float()
    if c["reverse"]:
        a, v = a.flip(1), v.flip(1)
    h0 = s["state"] if s["state"] is not None else torch.zeros((c["b"], c["d"]), device=v.device)
    prod, h = _doubling(a, v)
    h = h + prod * h0[:, None]
    out = {"h": (h.flip(1) if c["reverse"] else h).to(dt), "last": h[:, -1].clone()}
    if not c["train"]:
        return out
    g = s["d_h"].float()
    if c["reverse"]:
        g = g.flip(1)
    g = torch.cat([g[:, :-1], (g[:, -1] + s["d_last"])[:, None]], 1)
    # G[t] = g[t] + a[t+1] G[t+1]: the same recurrence from the far end, with the gates moved by one
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    _, G = _doubling(later.flip(1), g.flip(1))
    G = G.flip(1)
    before = torch.cat([h0[:, None], h[:, :-1]], 1)
    d_gate = G * before
    if c["gate"] == "shared":
        d_gate = d_gate.sum(2, keepdim=True)
    if c["reverse"]:
        d_gate, d_value = d_gate.flip(1), G.flip(1)
    else:
        d_value = G
    out["d_gate"], out["d_value"] = d_gate.to(dt), d_value.to(dt)
    if s["state"] is not None:
        out["d_state"] = a[:, 0] * G[:, 0]
    return out


# ----------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "group":
        n, g = case["n"], case["groups"]
        return {"bytes": 8 * n + 4 * n + 4 * (g + 1), "flops": n}
    e = BYTES[case["dtype"]]
    if op == "embed":
        n, r, d = case["n"], case["rows"], case["dim"]
        moved = 8 * n + e * (min(n, r) * d + n * d)
        if case["train"]:
            moved += e * (n * d + r * d)
        return {"bytes": moved, "flops": n * d * (2 if case["train"] else 1)}
    if op == "linear":
        n, g, k, m = case["n"], case["groups"], case["k"], case["m"]
        moved = 4 * n + e * (n * k + n * m + g * m * (k + 1))
        flops = 2 * n * k * m
        if case["train"]:
            moved += e * (n * m + n * k + g * m * (k + 1))
            flops *= 3
        return {"bytes": moved, "flops": flops}
    b, t, d = case["b"], case["t"], case["d"]
    gates = b * t * (1 if case["gate"] == "shared" else d)
    moved = e * (gates + 2 * b * t * d) + 4 * b * d * (2 if case["state"] else 1)
    flops = 2 * b * t * d
    if case["train"]:
        moved += e * (gates + 2 * b * t * d) + 4 * b * d * (2 if case["state"] else 1)
        flops *= 3
    return {"bytes": moved, "flops": flops}


# ----------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ----------------------------------------------------------------------------------------------------------------

@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "group":
        ids = s["ids"].cpu().tolist()
        buckets = [[] for _ in range(case["groups"] + 1)]
        for i, v in enumerate(ids):
            buckets[v if 0 <= v < case["groups"] else -1].append(i)
        offsets = [0]
        for bucket in buckets[:-1]:
            offsets.append(offsets[-1] + len(bucket))
        flat = [i for bucket in buckets for i in bucket]
        return {"order": torch.tensor(flat, dtype=torch.int32, device=DEV), "offsets": torch.tensor(offsets, dtype=torch.int32, device=DEV)}
    if op == "embed":
        ids, table = s["ids"], s["table"].double()
        padded = torch.cat([table, torch.zeros_like(table[:1])])              # one more row, of zeros, for ids of no row
        at = torch.where((ids < 0) | (ids >= case["rows"]), case["rows"], ids)
        out = {"out": padded[at] * s["scale"]}
        if case["train"]:
            grad = torch.zeros_like(padded)
            grad.index_add_(0, at, s["d_out"].double() * s["scale"])
            out["d_table"] = grad[:-1]
        return out
    if op == "linear":
        x, w, b, ids = (s[n].double() if n != "ids" else s[n] for n in ("x", "weight", "bias", "ids"))
        y = x.new_zeros((case["n"], case["m"]))
        dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
        for e in range(case["groups"]):
            rows = torch.nonzero(ids == e)[:, 0]
            xe = x.index_select(0, rows)
            z = torch.addmm(b[e][None], xe, w[e].t().contiguous())
            y.index_copy_(0, rows, z.clamp_min(0) if case["relu"] else z)
            if case["train"]:
                ge = s["d_out"].index_select(0, rows).double()
                dx.index_copy_(0, rows, torch.mm(ge, w[e]))
                dw[e] = torch.mm(ge.t().contiguous(), xe)
                db[e] = ge.sum(0)
        return {"y": y, "d_x": dx, "d_weight": dw, "d_bias": db} if case["train"] else {"y": y}
    return _exact_scan(case, s)


def _stepwise(a, v, h0):
    """h[t] = a[t] h[t-1] + v[t] in 64 bits: step by step inside pieces of about sqrt(T) samples, all pieces at once,
    then piece by piece, then every piece once more from its true state."""
    b, t, d = v.shape
    span = max(1, math.isqrt(t))
    pieces = (t + span - 1) // span
    pad = pieces * span - t
    if pad:                                                                     # gate 1, value 0 leave the state as it is
        a = torch.cat([a, a.new_ones((b, pad, a.shape[2]))], 1)
        v = torch.cat([v, v.new_zeros((b, pad, d))], 1)
    a, v = a.reshape(b, pieces, span, -1), v.reshape(b, pieces, span, d)
    end, gain = v.new_zeros((b, pieces, d)), torch.ones_like(a[:, :, 0])
    for i in range(span):
        end = a[:, :, i] * end + v[:, :, i]
        gain = gain * a[:, :, i]
    start = v.new_empty((b, pieces, d))
    h = h0
    for p in range(pieces):
        start[:, p] = h
        h = gain[:, p] * h + end[:, p]
    out = torch.empty_like(v)
    for i in range(span):
        start = a[:, :, i] * start + v[:, :, i]
        out[:, :, i] = start
    return out.reshape(b, pieces * span, d)[:, :t]


def _exact_scan(case, s):
    b, t, d = case["b"], case["t"], case["d"]
    a, v = s["gate"].double(), s["value"].double()
    h0 = s["state"].double() if s["state"] is not None else v.new_zeros((b, d))
    way = torch.arange(t - 1, -1, -1, device=DEV) if case["reverse"] else torch.arange(t, device=DEV)
    a, v = a[:, way], v[:, way]
    h = _stepwise(a, v, h0)
    out = {"h": h[:, way], "last": h[:, -1]}
    if not case["train"]:
        return out
    g = s["d_h"].double()[:, way].clone()
    g[:, -1] += s["d_last"].double()
    back = torch.arange(t - 1, -1, -1, device=DEV)
    moved = torch.ones_like(a)
    moved[:, 1:] = a[:, back[:-1]]                                              # gate of the sample that comes after
    total = _stepwise(moved, g[:, back], torch.zeros_like(h0))[:, back]
    prev = torch.empty_like(h)
    prev[:, 0], prev[:, 1:] = h0, h[:, :-1]
    d_gate = total * prev
    if case["gate"] == "shared":
        d_gate = d_gate.sum(-1, keepdim=True)
    out["d_gate"], out["d_value"] = d_gate[:, way], total[:, way]
    if s["state"] is not None:
        out["d_state"] = (a[:, 0] * total[:, 0])
    return out
