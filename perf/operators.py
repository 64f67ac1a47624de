"""Cases of the many-class loss and of rows sorted by expert.

Kinds of case:

- ``xent``: cross entropy of scores ``h W' + b`` over many classes
  (``mbk_xent``): each row's loss and log-sum-exp.
- ``xent_grad``: the same with the gradients of the summed loss by ``h``, ``W``
  and ``b`` (``mbk_xent_grad``).
- ``sort``: rows sorted by expert (``mbk_expert_sort``): offsets, the assignment
  in each slot and the slot of each assignment.
- ``dispatch``: the sort and the rows' features in that order
  (``mbk_expert_gather``).
- ``combine``: the experts' outputs back in the rows' order, weighted
  (``mbk_expert_combine``).
- ``combine_grad``: its gradients by the outputs and the weights
  (``mbk_expert_combine_grad``).
- ``dispatch_grad``: the gradient of ``dispatch`` by the features, which is
  ``mbk_expert_combine`` without weights.

``major`` is the layout of the rows' matrix (``row``: [rows][cols], ``feature``:
[cols][rows]); ``blocked`` says that the sorted matrix holds one feature-major
block [cols][rows of the expert] per expert, as the batch predictor takes it,
and not [slots][cols].
"""
import ctypes
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_CODES = {"f32": 0, "bf16": 1}


def listed():
    return [
        # The loss of one row while serving: launches and host steps are all there is.
        {"name": "xent_one", "kind": "xent", "type": "f32", "rows": 1, "dim": 64,
         "classes": 1000, "bias": True, "weighted": False, "out": 0.0, "masked": 0.0, "pad": 0},
        # A small request against a long list of classes: reading W is the work.
        {"name": "xent_serve_bf16", "kind": "xent", "type": "bf16", "rows": 16, "dim": 1024,
         "classes": 100000, "bias": False, "weighted": False, "out": 0.0, "masked": 0.0,
         "pad": 0},
        # Validation loss of a padded batch with an odd number of rows.
        {"name": "xent_eval_bf16", "kind": "xent", "type": "bf16", "rows": 8191, "dim": 768,
         "classes": 50000, "bias": True, "weighted": False, "out": 0.05, "masked": 0.0, "pad": 0},
        # One boosting round of 37 outputs for 1003 classes, sample weights, sizes that are
        # multiples of nothing.
        {"name": "xent_boost_odd", "kind": "xent_grad", "type": "f32", "rows": 99991, "dim": 37,
         "classes": 1003, "bias": True, "weighted": True, "out": 0.02, "masked": 0.05, "pad": 3},
        # The same with 100 outputs for 10000 classes on a 20k-row data set.
        {"name": "xent_boost_20k", "kind": "xent_grad", "type": "f32", "rows": 20000, "dim": 100,
         "classes": 10000, "bias": True, "weighted": True, "out": 0.0, "masked": 0.0, "pad": 0},
        # The largest: a training step on wide bf16 embeddings.
        {"name": "xent_step_bf16", "kind": "xent_grad", "type": "bf16", "rows": 16384,
         "dim": 1024, "classes": 65536, "bias": False, "weighted": True, "out": 0.01,
         "masked": 0.0, "pad": 0},
        # 10M rows to one of 1000 segments.
        {"name": "sort_10m", "kind": "sort", "rows": 10000000, "k": 1, "experts": 1000,
         "skew": 1.0, "dropped": 0.01},
        # A request of a thousand rows to four boosters.
        {"name": "dispatch_1k", "kind": "dispatch", "type": "f32", "rows": 1000, "cols": 10,
         "k": 1, "experts": 4, "major": "feature", "blocked": True, "skew": 0.0, "dropped": 0.0,
         "pad": 0},
        # 1M x 100 features to the boosters of 20 segments, each booster's rows as the
        # feature-major block that prediction and training take.
        {"name": "dispatch_1m", "kind": "dispatch", "type": "f32", "rows": 1000000, "cols": 100,
         "k": 1, "experts": 20, "major": "feature", "blocked": True, "skew": 1.0, "dropped": 0.0,
         "pad": 0},
        # 37 boosted outputs of the two best of five boosters, summed for each row.
        {"name": "combine_odd", "kind": "combine", "type": "f32", "rows": 99991, "cols": 37,
         "k": 2, "experts": 5, "major": "row", "blocked": True, "skew": 0.5, "dropped": 0.1,
         "pad": 3},
        # Wide bf16 rows to two of 64 experts, and the gradient of their way back.
        {"name": "dispatch_wide_bf16", "kind": "dispatch", "type": "bf16", "rows": 65536,
         "cols": 1024, "k": 2, "experts": 64, "major": "row", "blocked": False, "skew": 0.5,
         "dropped": 0.0, "pad": 0},
        {"name": "combine_grad_wide_bf16", "kind": "combine_grad", "type": "bf16", "rows": 65536,
         "cols": 1024, "k": 2, "experts": 64, "major": "row", "blocked": False, "skew": 0.5,
         "dropped": 0.0, "pad": 0},
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["xent", "xent", "xent_grad", "xent_grad", "xent_grad", "sort", "dispatch",
                       "dispatch", "combine", "combine", "combine_grad", "dispatch_grad"])
    case = {"kind": kind}
    if kind.startswith("xent"):
        case["type"] = rng.choice(["f32", "bf16"])
        dim = _spread(rng, 4, 1536)
        if dim > 32 and rng.random() < 0.6:
            dim -= dim % 32
        case["dim"] = dim
        case["classes"] = _spread(rng, 3, 131072)
        products = 1 << 40 if case["type"] == "bf16" else 1 << 36
        most = min(131072, (1 << 30) // case["classes"], products // (case["classes"] * dim))
        case["rows"] = _spread(rng, 1, max(1, most))
        case["bias"] = rng.random() < 0.6
        case["weighted"] = rng.random() < 0.5
        case["out"] = rng.choice([0.0, 0.0, 0.05, 0.5])
        case["masked"] = rng.choice([0.0, 0.0, 0.1]) if case["bias"] else 0.0
        case["pad"] = rng.choice([0, 0, 0, rng.randint(1, 24)])
        return case
    case["k"] = rng.choice([1, 1, 2, 2, 4, 8])
    case["experts"] = _spread(rng, 1, 4096)
    case["skew"] = rng.choice([0.0, 0.5, 1.0])
    case["dropped"] = rng.choice([0.0, 0.0, 0.05, 0.5])
    if kind == "sort":
        case["rows"] = _spread(rng, 1, 10000000 // case["k"])
        return case
    case["type"] = rng.choice(["f32", "bf16"])
    case["cols"] = _spread(rng, 1, 2048)
    elements = 1 << 27 if case["type"] == "bf16" else 1 << 26
    case["rows"] = _spread(rng, 1, min(2000000, max(1, elements // (case["cols"] * case["k"]))))
    case["major"] = rng.choice(["row", "row", "feature"])
    case["blocked"] = rng.random() < 0.5
    case["pad"] = rng.choice([0, 0, 0, rng.randint(1, 24)])
    return case


# ---- inputs -----------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _matrix(gen, rows, cols, case, scale=1.0):
    """[rows][cols] of normal values, with pad elements between the rows of memory."""
    full = torch.empty((rows, cols + case["pad"]), device="cuda").normal_(generator=gen)
    return full.mul_(scale).to(_TYPES[case["type"]])[:, :cols]


def _blank(rows, cols, case):
    return torch.zeros((rows, cols + case["pad"]), device="cuda",
                       dtype=_TYPES[case["type"]])[:, :cols]


def _prepare_xent(case, gen):
    n, d, v = case["rows"], case["dim"], case["classes"]
    s = {"h": _matrix(gen, n, d, case), "w": _matrix(gen, v, d, case, 2.0 / math.sqrt(d)),
         "bias": None, "weights": None}
    open_classes = torch.arange(v, device="cuda")
    if case["bias"]:
        s["bias"] = torch.empty(v, device="cuda").normal_(generator=gen).mul_(0.5)
        if case["masked"] > 0:
            closed = torch.rand(v, generator=gen, device="cuda") < case["masked"]
            closed[0] = False
            s["bias"][closed] = -math.inf
            open_classes = open_classes[~closed]
    pick = torch.randint(open_classes.numel(), (n,), generator=gen, device="cuda")
    s["labels"] = open_classes[pick].int()
    if case["out"] > 0:
        s["labels"][torch.rand(n, generator=gen, device="cuda") < case["out"]] = -1
    if case["weighted"]:
        s["weights"] = torch.rand(n, generator=gen, device="cuda") + 0.5
    if own:
        s["loss"] = torch.zeros(n, device="cuda")
        s["lse"] = torch.zeros(n, device="cuda")
        if case["kind"] == "xent_grad":
            s["dh"], s["dw"] = _blank(n, d, case), _blank(v, d, case)
            s["db"] = torch.zeros(v, device="cuda") if case["bias"] else None
    return s


def _prepare_experts(case, gen):
    n, k, e = case["rows"], case["k"], case["experts"]
    popular = torch.arange(1, e + 1, device="cuda", dtype=torch.float64) ** -case["skew"]
    share = torch.cumsum(popular, 0) / popular.sum()
    u = torch.rand((n, k), generator=gen, device="cuda", dtype=torch.float64)
    expert = torch.searchsorted(share, u).clamp_(max=e - 1)
    expert = ((expert * 7 + 3) % e if e % 7 else expert).int()
    if case["dropped"] > 0:
        expert[torch.rand((n, k), generator=gen, device="cuda") < case["dropped"]] = -1
    s = {"expert": expert}
    slots = n * k
    if case["kind"] in ("sort", "dispatch"):
        if own:
            s["offsets"] = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
            s["source"] = torch.zeros(slots, dtype=torch.int32, device="cuda")
            s["slot"] = torch.zeros((n, k), dtype=torch.int32, device="cuda")
    else:
        s["offsets"], s["source"], s["slot"] = _plain_sort(expert, e)
    if case["kind"] == "sort":
        return s
    cols, dtype = case["cols"], _TYPES[case["type"]]

    def rows_matrix(values):
        if case["major"] == "row":
            return _matrix(gen, n, cols, case) if values else _blank(n, cols, case)
        return (_matrix(gen, cols, n, case) if values else _blank(cols, n, case)).T

    if case["kind"] == "dispatch":
        s["x"] = rows_matrix(True)
        if own:
            s["sorted"] = torch.zeros(slots * cols, dtype=dtype, device="cuda")
        return s
    s["y"] = torch.empty(slots * cols, device="cuda").normal_(generator=gen).to(dtype)
    s["weights"] = None
    if case["kind"] != "dispatch_grad":
        gate = torch.empty((n, k), device="cuda").normal_(generator=gen)
        s["weights"] = torch.exp(gate) / torch.exp(gate).sum(1, keepdim=True)
    if case["kind"] == "combine_grad":
        s["dout"] = rows_matrix(True)
        if own:
            s["dy"] = torch.zeros(slots * cols, dtype=dtype, device="cuda")
            s["dweights"] = torch.zeros((n, k), device="cuda")
    elif own:
        s["out"] = rows_matrix(False)
    return s


def prepare(case, seed):
    gen = _generator(seed)
    s = _prepare_xent(case, gen) if case["kind"].startswith("xent") else _prepare_experts(case, gen)
    s["case"] = case
    if own:
        _describe(s)
    torch.cuda.synchronize()
    return s


# ---- the plain forms ----------------------------------------------------------

_SCORES = 1 << 30       # scores held at a time: more rows go in turns


def _plain_xent(s, grad):
    h, w, bias, labels, weights = s["h"], s["w"], s["bias"], s["labels"], s["weights"]
    n, v = h.shape[0], w.shape[0]
    wf = w.float()
    wt = wf.T.contiguous()
    if bias is None:
        bias = torch.zeros(v, device=h.device)
    if weights is None:
        weights = torch.ones(n, device=h.device)
    weights = torch.where((labels >= 0) & (labels < v), weights, torch.zeros_like(weights))
    at = labels.long().clamp(0, v - 1)[:, None]
    loss, lse = torch.empty(n, device=h.device), torch.empty(n, device=h.device)
    if grad:
        dh = torch.empty(h.shape, device=h.device)
        dw, db = torch.zeros(w.shape, device=h.device), torch.zeros(v, device=h.device)
    step = max(1, _SCORES // v)
    for a in range(0, n, step):
        r = slice(a, min(n, a + step))
        hf = h[r].float()
        z = hf @ wt + bias
        top = z.max(1, keepdim=True).values
        p = torch.exp(z - top)
        total = p.sum(1, keepdim=True)
        lse[r] = (top + torch.log(total))[:, 0]
        # 0 for a row that is out, whatever its scores
        value = lse[r] - z.gather(1, at[r])[:, 0]
        loss[r] = torch.where(weights[r] != 0, weights[r] * value, torch.zeros_like(value))
        if grad:
            p /= total
            p.scatter_add_(1, at[r], torch.full_like(lse[r], -1.0)[:, None])
            p *= weights[r][:, None]
            dh[r] = p @ wf
            dw += p.T @ hf
            db += p.sum(0)
    if not grad:
        return loss, lse
    out = [loss, lse, dh.to(h.dtype), dw.to(w.dtype)]
    return out + [db] if s["bias"] is not None else out


def _plain_sort(expert, experts):
    flat = expert.flatten().long()
    key = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
    ordered, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(ordered, torch.arange(experts + 1, device=flat.device))
    here = torch.arange(flat.numel(), device=flat.device)
    kept = ordered < experts
    source = torch.where(kept, order, torch.full_like(order, -1))
    slot = torch.empty_like(order)
    slot[order] = torch.where(kept, here, torch.full_like(here, -1))
    return offsets.int(), source.int(), slot.int().reshape(expert.shape)


def _places(offsets, source, experts, cols, blocked):
    """Where element (slot, column) lies in the sorted matrix, and which slots are taken."""
    slots = source.numel()
    at = torch.arange(slots, device=source.device)
    col = torch.arange(cols, device=source.device)
    if not blocked:
        return at[:, None] * cols + col, source >= 0
    off = offsets.long()
    e = (torch.searchsorted(off, at, right=True) - 1).clamp(0, experts - 1)
    size = off[e + 1] - off[e]
    return off[e][:, None] * cols + col * size[:, None] + (at - off[e])[:, None], source >= 0


def _plain_dispatch(s):
    case = s["case"]
    offsets, source, slot = _plain_sort(s["expert"], case["experts"])
    place, taken = _places(offsets, source, case["experts"], case["cols"], case["blocked"])
    rows = source[taken].long() // case["k"]
    out = torch.zeros(source.numel() * case["cols"], dtype=s["x"].dtype, device=s["x"].device)
    out[place[taken]] = s["x"][rows]
    return offsets, source, slot, out


def _plain_combine(s):
    case = s["case"]
    place, _ = _places(s["offsets"], s["source"], case["experts"], case["cols"], case["blocked"])
    out = torch.zeros((case["rows"], case["cols"]), device=s["y"].device)
    for j in range(case["k"]):
        at = s["slot"][:, j].long()
        term = s["y"][place[at.clamp(min=0)]].float()
        if s["weights"] is not None:
            term = term * s["weights"][:, j:j + 1]
        out += torch.where(at[:, None] >= 0, term, torch.zeros_like(term))
    return out.to(s["y"].dtype)


def _plain_combine_grad(s):
    case = s["case"]
    place, _ = _places(s["offsets"], s["source"], case["experts"], case["cols"], case["blocked"])
    dy = torch.zeros_like(s["y"])
    dweights = torch.zeros((case["rows"], case["k"]), device=dy.device)
    dout = s["dout"].float()
    for j in range(case["k"]):
        at = s["slot"][:, j].long()
        kept = at >= 0
        y = s["y"][place[at.clamp(min=0)]].float()
        dweights[:, j] = torch.where(kept, (dout * y).sum(1), torch.zeros_like(dweights[:, j]))
        dy[place[at[kept]]] = (dout[kept] * s["weights"][kept, j:j + 1]).to(dy.dtype)
    return dy, dweights


# ---- the framework's operators ------------------------------------------------

_contexts = {}


def _context():
    """The context on the current stream, kept as a program keeps it."""
    import macboost_amd as mb
    key = (torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream)
    if key not in _contexts:
        _contexts[key] = mb.Context(key[0], stream=key[1])
    return _contexts[key]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _describe(s):
    """The structures that describe the buffers to the library."""
    from macboost_amd import _core
    case = s["case"]
    _context()
    if case["kind"].startswith("xent"):
        s["shape"] = _core.MbkXentShape(case["rows"], case["classes"], case["dim"],
                                        _CODES[case["type"]], s["h"].stride(0), s["w"].stride(0))
        return
    s["plan"] = _core.MbkExpertPlan(case["rows"], case["k"], case["experts"], _ptr(s["expert"]),
                                    _ptr(s["offsets"]), _ptr(s["source"]), _ptr(s["slot"]))
    for name in ("x", "out", "dout"):
        if name in s:
            s["matrix"] = _core.MbkExpertMatrix(
                _ptr(s[name]), s[name].stride(0), s[name].stride(1), case["cols"],
                _CODES[case["type"]], int(case["blocked"]))


def _own_run(s):
    ctx, kind = _context(), s["case"]["kind"]
    ref = ctypes.byref
    if kind.startswith("xent"):
        inputs = (ref(s["shape"]), _ptr(s["h"]), _ptr(s["w"]), _ptr(s["bias"]), _ptr(s["labels"]),
                  _ptr(s["weights"]), _ptr(s["loss"]), _ptr(s["lse"]))
        if kind == "xent":
            ctx.call("mbk_xent", *inputs)
            return s["loss"], s["lse"]
        ctx.call("mbk_xent_grad", *inputs, _ptr(s["dh"]), _ptr(s["dw"]), _ptr(s["db"]))
        out = [s["loss"], s["lse"], s["dh"], s["dw"]]
        return out + [s["db"]] if s["db"] is not None else out
    if kind in ("sort", "dispatch"):
        ctx.call("mbk_expert_sort", ref(s["plan"]))
        order = (s["offsets"], s["source"], s["slot"])
        if kind == "sort":
            return order
        ctx.call("mbk_expert_gather", ref(s["plan"]), ref(s["matrix"]), _ptr(s["sorted"]))
        return order + (s["sorted"],)
    if kind == "combine_grad":
        ctx.call("mbk_expert_combine_grad", ref(s["plan"]), ref(s["matrix"]), _ptr(s["y"]),
                 _ptr(s["weights"]), _ptr(s["dy"]), _ptr(s["dweights"]))
        return s["dy"], s["dweights"]
    ctx.call("mbk_expert_combine", ref(s["plan"]), _ptr(s["y"]), _ptr(s["weights"]),
             ref(s["matrix"]))
    return s["out"]


def run(state):
    if own:
        return _own_run(state)
    kind = state["case"]["kind"]
    if kind.startswith("xent"):
        return _plain_xent(state, kind == "xent_grad")
    if kind == "sort":
        return _plain_sort(state["expert"], state["case"]["experts"])
    if kind == "dispatch":
        return _plain_dispatch(state)
    if kind == "combine_grad":
        return _plain_combine_grad(state)
    return _plain_combine(state)


# ---- the work -------------------------------------------------------------------

def work(case):
    n = case["rows"]
    size = 4 if case.get("type") == "f32" else 2
    if case["kind"].startswith("xent"):
        d, v = case["dim"], case["classes"]
        moved = (n + v) * d * size + 12 * n
        if case["bias"]:
            moved += 4 * v
        if case["weighted"]:
            moved += 4 * n
        if case["kind"] == "xent":
            return {"bytes": moved, "flops": 2 * n * d * v}
        moved += (n + v) * d * size + (4 * v if case["bias"] else 0)
        return {"bytes": moved, "flops": 6 * n * d * v}
    slots = n * case["k"]
    kept = slots * (1 - case["dropped"])
    sort = 12 * slots + 4 * (case["experts"] + 1)
    if case["kind"] == "sort":
        return {"bytes": sort, "flops": 0}
    rows, placed = n * case["cols"] * size, int(kept * case["cols"] * size)
    if case["kind"] == "dispatch":
        return {"bytes": sort + rows + placed, "flops": 0}
    if case["kind"] == "combine_grad":
        return {"bytes": rows + 2 * placed + 12 * slots, "flops": int(3 * kept * case["cols"])}
    moved = rows + placed + 4 * slots
    if case["kind"] == "dispatch_grad":
        return {"bytes": moved, "flops": int(kept * case["cols"])}
    return {"bytes": moved + 4 * slots, "flops": int(2 * kept * case["cols"])}


# ---- from the definitions, in 64 bits ---------------------------------------------

def _exact_xent(s, grad):
    n, v = s["h"].shape[0], s["w"].shape[0]
    w = s["w"].double()
    loss = torch.zeros(n, dtype=torch.float64, device=w.device)
    lse = torch.zeros_like(loss)
    dh = torch.zeros(s["h"].shape, dtype=torch.float64, device=w.device)
    dw = torch.zeros_like(w)
    db = torch.zeros(v, dtype=torch.float64, device=w.device)
    for a in range(0, n, max(1, (1 << 28) // v)):
        b = min(n, a + max(1, (1 << 28) // v))
        h = s["h"][a:b].double()
        z = torch.mm(h, w.t())
        if s["bias"] is not None:
            z += s["bias"].double()
        lse[a:b] = torch.logsumexp(z, 1)
        y = s["labels"][a:b].long()
        inside = (y >= 0) & (y < v)
        scale = inside.double()
        if s["weights"] is not None:
            scale *= s["weights"][a:b].double()
        rows = torch.nonzero(inside)[:, 0]
        loss[a:b][rows] = scale[rows] * (lse[a:b][rows] - z[rows, y[rows]])
        if grad:
            g = torch.exp(z - lse[a:b, None])
            g[rows, y[rows]] -= 1
            g *= scale[:, None]
            dh[a:b] = torch.mm(g, w)
            dw += torch.mm(g.t().contiguous(), h)
            db += g.sum(0)
    if not grad:
        return loss, lse
    out = [loss, lse, dh, dw]
    return out + [db] if s["bias"] is not None else out


def _exact_sort(expert, experts):
    flat = expert.cpu().numpy().ravel()
    kept = np.flatnonzero((flat >= 0) & (flat < experts))
    order = kept[np.argsort(flat[kept].astype(np.uint16), kind="stable")]
    source = np.full(flat.size, -1, np.int32)
    source[:order.size] = order
    slot = np.full(flat.size, -1, np.int32)
    slot[order] = np.arange(order.size)
    offsets = np.zeros(experts + 1, np.int32)
    offsets[1:] = np.cumsum(np.bincount(flat[kept], minlength=experts))
    return offsets, source, slot.reshape(tuple(expert.shape))


def _exact_blocks(offsets, cols, case):
    """(first slot, rows, first element) of each expert's part of the sorted matrix."""
    return [(int(a), int(b - a), int(a) * cols) for a, b in zip(offsets[:-1], offsets[1:])]


def _sorted_rows(flat, offsets, cols, case):
    """The sorted matrix as [slots][cols], whatever its layout."""
    if not case["blocked"]:
        return flat.reshape(-1, cols)
    out = torch.zeros_like(flat).reshape(-1, cols)
    for first, size, begin in _exact_blocks(offsets, cols, case):
        if size:
            out[first:first + size] = flat[begin:begin + size * cols].reshape(cols, size).t()
    return out


def _sorted_flat(rows, offsets, cols, case):
    if not case["blocked"]:
        return rows.reshape(-1)
    out = torch.zeros_like(rows).reshape(-1)
    for first, size, begin in _exact_blocks(offsets, cols, case):
        if size:
            out[begin:begin + size * cols] = rows[first:first + size].t().reshape(-1)
    return out


def _exact_experts(s):
    case = s["case"]
    order = _exact_sort(s["expert"], case["experts"])
    offsets, source, slot = order
    if case["kind"] == "sort":
        return order
    cols, k, kept = case["cols"], case["k"], int(offsets[-1])
    which = torch.from_numpy(source[:kept].astype(np.int64)).cuda()
    if case["kind"] == "dispatch":
        rows = torch.zeros((source.size, cols), dtype=torch.float64, device="cuda")
        rows[:kept] = s["x"].double()[which // k]
        return order + (_sorted_flat(rows, offsets, cols, case),)
    y = _sorted_rows(s["y"].double(), offsets, cols, case)
    weight = torch.ones((case["rows"], k), dtype=torch.float64, device="cuda")
    if s["weights"] is not None:
        weight = s["weights"].double()
    if case["kind"] == "combine_grad":
        dout = s["dout"].double()[which // k]
        dy = torch.zeros_like(y)
        dy[:kept] = dout * weight.reshape(-1)[which][:, None]
        dweights = torch.zeros(case["rows"] * k, dtype=torch.float64, device="cuda")
        dweights[which] = (dout * y[:kept]).sum(1)
        return _sorted_flat(dy, offsets, cols, case), dweights.reshape(case["rows"], k)
    out = torch.zeros((case["rows"], cols), dtype=torch.float64, device="cuda")
    out.index_add_(0, which // k, y[:kept] * weight.reshape(-1)[which][:, None])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"].startswith("xent"):
        return _exact_xent(s, case["kind"] == "xent_grad")
    return _exact_experts(s)
