"""Cases of category vectors beside the forests, of clipping many gradients and of answers with
class vectors in 4 bits.

Kinds of case:

- ``embed``: each row's category vector, scaled, on top of what the forests gave
  (``mbk_embed``).
- ``embed_grad``: the gradient of the category vectors (``mbk_embed_grad``).
- ``clip``: the norm of many gradients together, and each of them scaled so that it is at most
  ``max_norm`` (``mbk_grad_clip``).
- ``scores``: the classes' scores ``h W' + b`` with W in 4 bits and a scale for each group of
  ``group`` elements of a class (``mbk_fourbit_scores``).
- ``adjust``: scores with penalties for the classes that a row's history holds, biases, and -inf for
  classes that are not allowed (``mbk_adjust``).

W in 4 bits: a group's scale is bf16(max |w| * f32(1/7)), an element's code the whole number nearest
to w / scale, ties to even, in -8..7 (0 where the scale is 0); it stands for code * scale.
"""
import ctypes
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_CODES = {"f32": 0, "bf16": 1}
_SEVENTH = float(np.float32(1 / 7))


def _f32(value):
    """The value as the library's float arguments hold it."""
    return float(np.float32(value))


def listed():
    return [
        # A request of a few rows: one launch is all there is.
        {"name": "embed_request", "kind": "embed", "type": "f32", "rows": 64, "dim": 37,
         "entries": 1003, "base": True, "skew": 1.0, "dropped": 0.05, "pad": 3, "scale": 1.0},
        # The vectors of a column of a million categories for a batch, added to wide bf16 rows.
        {"name": "embed_wide_bf16", "kind": "embed", "type": "bf16", "rows": 65536, "dim": 1024,
         "entries": 100000, "base": True, "skew": 0.5, "dropped": 0.0, "pad": 0, "scale": 0.25},
        # 37 outputs, a few hundred categories, a data set of 99991 rows: long sums.
        {"name": "embed_grad_odd", "kind": "embed_grad", "type": "f32", "rows": 99991, "dim": 37,
         "entries": 300, "base": False, "skew": 0.5, "dropped": 0.02, "pad": 3, "scale": 1.0},
        # A million rows of 64 outputs, 100000 categories of which few are common.
        {"name": "embed_grad_1m", "kind": "embed_grad", "type": "f32", "rows": 1000000,
         "dim": 64, "entries": 100000, "base": False, "skew": 1.0, "dropped": 0.0, "pad": 0,
         "scale": 1.0},
        # A training step on wide bf16 embeddings, on top of the gradient that is there.
        {"name": "embed_grad_wide_bf16", "kind": "embed_grad", "type": "bf16", "rows": 16384,
         "dim": 1024, "entries": 65536, "base": True, "skew": 0.5, "dropped": 0.01, "pad": 0,
         "scale": 0.25},
        # The gradients of a small many-class model: its class vectors, biases, a few tables.
        {"name": "clip_small", "kind": "clip", "type": "f32", "tensors": 6, "rows": 1003,
         "cols": 37, "shrink": 1.0, "pad": 3, "ratio": 0.5},
        # A table for each of 200 columns, class vectors and biases, both types.
        {"name": "clip_many", "kind": "clip", "type": "mixed", "tensors": 200, "rows": 100000,
         "cols": 64, "shrink": 0.5, "pad": 0, "ratio": 0.5},
        # One row answered by a small model.
        {"name": "scores_one", "kind": "scores", "type": "f32", "rows": 1, "dim": 64,
         "classes": 1000, "group": 32, "bias": True, "masked": 0.0, "pad": 0},
        # A small request against a long list of classes: reading W is the work.
        {"name": "scores_serve_bf16", "kind": "scores", "type": "bf16", "rows": 16, "dim": 1024,
         "classes": 100000, "group": 128, "bias": False, "masked": 0.0, "pad": 0},
        # A ragged batch in f32 with small groups, some classes not offered.
        {"name": "scores_batch_odd", "kind": "scores", "type": "f32", "rows": 201, "dim": 777,
         "classes": 50003, "group": 32, "bias": True, "masked": 0.05, "pad": 3},
        # One row's scores under its history.
        {"name": "adjust_one", "kind": "adjust", "rows": 1, "classes": 1003, "history": 20,
         "ragged": False, "bias": True, "mask": "row", "allowed": 0.9, "pad": 1,
         "repetition": 1.2, "presence": 0.0, "frequency": 0.0},
        # A batch of requests with long histories, each with its own allowed classes.
        {"name": "adjust_batch", "kind": "adjust", "rows": 256, "classes": 100000,
         "history": 2000, "ragged": True, "bias": True, "mask": "row", "allowed": 0.5, "pad": 0,
         "repetition": 1.1, "presence": 0.5, "frequency": 0.1},
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["embed", "embed", "embed_grad", "embed_grad", "embed_grad", "clip", "clip",
                       "scores", "scores", "scores", "adjust", "adjust"])
    case = {"kind": kind}
    if kind in ("embed", "embed_grad"):
        case["type"] = rng.choice(["f32", "bf16"])
        dim = _spread(rng, 1, 2048)
        if dim > 16 and rng.random() < 0.6:
            dim -= dim % 16
        case["dim"] = dim
        most = (1 << 26) // dim
        case["entries"] = _spread(rng, 1, min(2000000, most))
        case["rows"] = _spread(rng, 1, min(1000000, most))
        case["base"] = rng.random() < 0.4
        case["skew"] = rng.choice([0.0, 0.5, 1.0, 1.5])
        case["dropped"] = rng.choice([0.0, 0.0, 0.05, 0.5]) if case["rows"] >= 64 else 0.0
        case["pad"] = rng.choice([0, 0, 0, rng.randint(1, 24)])
        case["scale"] = rng.choice([1.0, 0.25, round(rng.uniform(0.05, 32.0), 3)])
        return case
    if kind == "clip":
        case["type"] = rng.choice(["f32", "bf16", "mixed"])
        case["tensors"] = _spread(rng, 1, 500)
        case["cols"] = _spread(rng, 1, 2048)
        case["shrink"] = rng.choice([0.0, 0.5, 1.0])
        most = (1 << 27) // case["cols"]
        if case["shrink"] == 0.0:
            most //= case["tensors"]
        elif case["shrink"] == 0.5:
            most = int(most / (2 * math.sqrt(case["tensors"])))
        else:
            most = int(most / (1 + math.log(case["tensors"])))
        case["rows"] = _spread(rng, 1, max(1, min(500000, most)))
        case["pad"] = rng.choice([0, 0, 0, rng.randint(1, 24)])
        case["ratio"] = rng.choice([0.0, 0.1, 0.5, 0.5, 2.0])
        return case
    if kind == "scores":
        case["type"] = rng.choice(["f32", "bf16"])
        dim = _spread(rng, 8, 4096)
        if dim > 32 and rng.random() < 0.6:
            dim -= dim % 32
        case["dim"] = dim
        case["classes"] = _spread(rng, 3, min(200000, (1 << 27) // dim))
        most = min(512, (1 << 24) // case["classes"], (1 << 34) // (case["classes"] * dim))
        case["rows"] = _spread(rng, 1, max(1, most))
        case["group"] = rng.choice([32, 64, 128])
        case["bias"] = rng.random() < 0.6
        case["masked"] = rng.choice([0.0, 0.0, 0.1]) if case["bias"] else 0.0
        case["pad"] = rng.choice([0, 0, 0, rng.randint(1, 24)])
        return case
    case["classes"] = _spread(rng, 16, 200000)
    case["rows"] = _spread(rng, 1, min(1024, (1 << 25) // case["classes"]))
    case["history"] = rng.choice([0, _spread(rng, 1, 4000), _spread(rng, 1, 4000)])
    case["ragged"] = rng.random() < 0.5
    case["bias"] = rng.random() < 0.5
    case["mask"] = rng.choice(["none", "one", "row", "row"])
    case["allowed"] = rng.choice([0.5, 0.9, 0.999])
    case["pad"] = rng.choice([0, 0, 0, rng.randint(1, 24)])
    case["repetition"] = rng.choice([1.0, 1.2, 0.8])
    case["presence"] = rng.choice([0.0, 0.5, -0.25])
    case["frequency"] = rng.choice([0.0, 0.1, 0.7])
    return case


# ---- inputs -----------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _matrix(gen, rows, cols, pad, dtype, scale=1.0):
    """[rows][cols] of normal values, pad elements between the rows."""
    full = torch.empty((rows, cols + pad), device="cuda").normal_(generator=gen)
    return full.mul_(scale).to(dtype)[:, :cols]


def _blank(rows, cols, pad, dtype):
    return torch.zeros((rows, cols + pad), device="cuda", dtype=dtype)[:, :cols]


def _ids(gen, rows, count, skew, shape):
    """Ids of [0, count), popular in proportion to 1 / rank ** skew, ranks in no order."""
    share = torch.cumsum(torch.arange(1, count + 1, device="cuda",
                                      dtype=torch.float64) ** -skew, 0)
    u = torch.rand(shape, generator=gen, device="cuda", dtype=torch.float64) * share[-1]
    rank = torch.searchsorted(share, u).clamp_(max=count - 1)
    return torch.randperm(count, generator=gen, device="cuda")[rank].int()


def _prepare_embed(case, gen):
    n, d, e, dtype = case["rows"], case["dim"], case["entries"], _TYPES[case["type"]]
    s = {"ids": _ids(gen, n, e, case["skew"], (n,)), "base": None}
    if case["dropped"] > 0:
        s["ids"][torch.rand(n, generator=gen, device="cuda") < case["dropped"]] = -1
    if case["kind"] == "embed":
        s["table"] = _matrix(gen, e, d, case["pad"], dtype)
    else:
        s["dout"] = _matrix(gen, n, d, case["pad"], dtype)
    rows = n if case["kind"] == "embed" else e
    if case["base"]:
        s["base"] = _matrix(gen, rows, d, case["pad"], dtype)
    if own:
        s["out"] = _blank(rows, d, case["pad"], dtype)
    return s


def _tensor_shapes(case):
    """(rows, cols, type) of each gradient: matrices that get shorter, every third a vector."""
    out = []
    for i in range(case["tensors"]):
        rows = max(1, int(case["rows"] * (i + 1) ** -case["shrink"]))
        kind = case["type"] if case["type"] != "mixed" else ("bf16", "f32")[i % 2]
        out.append((1, rows, "f32") if i % 3 == 2 else (rows, case["cols"], kind))
    return out


def _layout(case):
    """Where each gradient lies in one buffer a type, as buckets of gradients lie: (type, first
    element, rows, cols), and the elements of each buffer."""
    places, size = [], {}
    for rows, cols, kind in _tensor_shapes(case):
        at = size.get(kind, 0)
        places.append((kind, at, rows, cols))
        size[kind] = at + (rows * (cols + case["pad"]) + 63) // 64 * 64
    return places, size


def _views(case, buffers):
    return [buffers[t][at:at + r * (c + case["pad"])].view(r, c + case["pad"])[:, :c]
            for t, at, r, c in _layout(case)[0]]


def _prepare_clip(case, gen):
    places, size = _layout(case)
    held = {t: torch.zeros(n, device="cuda", dtype=_TYPES[t]) for t, n in size.items()}
    s = {"grads": _views(case, held), "held": held, "buffers": None, "outs": []}
    for g in s["grads"]:
        g.copy_(torch.empty(g.shape, device="cuda").normal_(generator=gen).mul_(0.01))
    s["max_norm"] = math.inf
    if case["ratio"]:
        elements = sum(r * c for _, _, r, c in places)
        s["max_norm"] = _f32(case["ratio"] * 0.01 * math.sqrt(elements))
        s["buffers"] = {t: torch.zeros_like(x) for t, x in held.items()}
        s["outs"] = _views(case, s["buffers"])
    if own:
        s["norm"] = torch.zeros(1, device="cuda")
    return s


def _quantise(w, group):
    """Codes and scales of W, [classes][groups * group] and [classes][groups]."""
    v, d = w.shape
    groups = (d + group - 1) // group
    full = torch.zeros((v, groups * group), device=w.device)
    full[:, :d] = w.float()
    full = full.view(v, groups, group)
    scale = (full.abs().amax(2) * _SEVENTH).bfloat16()
    by = scale.float()[:, :, None]
    code = torch.where(by > 0, torch.round(full / by), torch.zeros_like(full))
    return code.clamp_(-8, 7).to(torch.int8).view(v, groups * group), scale


def _prepare_scores(case, gen):
    n, d, v, dtype = case["rows"], case["dim"], case["classes"], _TYPES[case["type"]]
    s = {"h": _matrix(gen, n, d, case["pad"], dtype), "bias": None}
    w = _matrix(gen, v, d, 0, dtype, 2.0 / math.sqrt(d))
    if case["bias"]:
        s["bias"] = torch.empty(v, device="cuda").normal_(generator=gen).mul_(0.5)
        if case["masked"] > 0:
            s["bias"][torch.rand(v, generator=gen, device="cuda") < case["masked"]] = -math.inf
    if own:
        s["w"] = w
        s["scores"] = _blank(n, v, case["pad"], torch.float32)
    else:
        code, s["scale"] = _quantise(w, case["group"])
        nibbles = (code + 8).to(torch.uint8)
        s["nibbles"] = nibbles[:, ::2] | (nibbles[:, 1::2] << 4)
    return s


def _prepare_adjust(case, gen):
    n, v, most = case["rows"], case["classes"], case["history"]
    s = {"scores": _matrix(gen, n, v, case["pad"], torch.float32, 3.0),
         "history": _ids(gen, n, v, 1.0, (n, max(1, most)))[:, :most].contiguous(),
         "lengths": None, "bias": None, "allowed": None}
    if case["ragged"]:
        s["lengths"] = torch.randint(most + 1, (n,), generator=gen, device="cuda").int()
    if case["bias"]:
        s["bias"] = torch.empty(v, device="cuda").normal_(generator=gen)
    if case["mask"] != "none":
        rows, words = (n if case["mask"] == "row" else 1), (v + 31) // 32
        s["allowed"] = torch.zeros((rows, words), dtype=torch.int32, device="cuda")
        for bit in range(32):
            on = torch.rand((rows, words), generator=gen, device="cuda") < case["allowed"]
            value = 1 << bit if bit < 31 else -(1 << 31)
            s["allowed"] |= torch.where(on, value, 0).int()
    if own:
        s["out"] = _blank(n, v, case["pad"], torch.float32)
    return s


def prepare(case, seed):
    gen = _generator(seed)
    s = {"embed": _prepare_embed, "embed_grad": _prepare_embed, "clip": _prepare_clip,
         "scores": _prepare_scores, "adjust": _prepare_adjust}[case["kind"]](case, gen)
    s["case"] = case
    if own:
        _describe(s)
    torch.cuda.synchronize()
    return s


# ---- the plain forms ----------------------------------------------------------

def _plain_embed(s):
    entries = s["case"]["entries"]
    ids = s["ids"].long()
    kept = (ids >= 0) & (ids < entries)
    out = s["table"][ids.clamp(0, entries - 1)].float() * _f32(s["case"]["scale"])
    out = torch.where(kept[:, None], out, torch.zeros_like(out))
    if s["base"] is not None:
        out += s["base"].float()
    return out.to(s["table"].dtype)


def _plain_embed_grad(s):
    case, dout = s["case"], s["dout"]
    ids = s["ids"].long()
    kept = (ids >= 0) & (ids < case["entries"])
    key, order = torch.sort(torch.where(kept, ids, torch.full_like(ids, case["entries"])))
    until = torch.searchsorted(key, torch.arange(case["entries"], device=key.device), right=True)
    # running sums of the rows in that order, in blocks and over the blocks
    n, d, step = ids.numel(), case["dim"], 256
    run = torch.zeros(((n + step - 1) // step, step, d), dtype=torch.float64, device=key.device)
    run.view(-1, d)[:n] = torch.where(kept[order][:, None], dout[order].double(), 0.0)
    run = torch.cumsum(run, 1)
    run[1:] += torch.cumsum(run[:-1, -1], 0)[:, None]
    run = torch.cat((run.new_zeros((1, d)), run.view(-1, d)))
    total = run[until]
    total[1:] -= run[until[:-1]]
    total *= _f32(case["scale"])
    if s["base"] is not None:
        total += s["base"].double()
    return total.to(dout.dtype)


def _plain_clip(s):
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    for g in s["grads"]:
        total += (g.double() ** 2).sum()
    norm = torch.sqrt(total)
    if math.isinf(s["max_norm"]):
        return [norm.float()[None]]
    by = torch.where(norm > s["max_norm"], s["max_norm"] / norm, torch.ones_like(norm)).float()
    for g, out in zip(s["grads"], s["outs"]):
        out.copy_(g.float() * by)
    return [norm.float()[None]] + list(s["buffers"].values())


def _plain_scores(s):
    case = s["case"]
    v, d, group = case["classes"], case["dim"], case["group"]
    code = torch.stack((s["nibbles"] & 15, s["nibbles"] >> 4), 2).view(v, -1, group).float() - 8
    w = (code * s["scale"].float()[:, :, None]).view(v, -1)[:, :d]
    z = s["h"].float() @ w.T.contiguous()
    return z if s["bias"] is None else z + s["bias"]


def _plain_adjust(s):
    case, z = s["case"], s["scores"]
    n, v = z.shape
    at = torch.arange(s["history"].shape[1], device=z.device)
    taken = (s["history"] >= 0) & (s["history"] < v)
    if s["lengths"] is not None:
        taken &= at[None, :] < s["lengths"][:, None]
    count = torch.zeros((n, v), device=z.device)
    count.scatter_add_(1, s["history"].long().clamp(0, v - 1), taken.float())
    seen = torch.where(z > 0, z / case["repetition"], z * case["repetition"])
    seen = seen - (case["presence"] + case["frequency"] * count)
    out = torch.where(count > 0, seen, z)
    if s["bias"] is not None:
        out = out + s["bias"]
    if s["allowed"] is not None:
        bits = torch.arange(32, device=z.device, dtype=torch.int32)
        on = ((s["allowed"][:, :, None] >> bits) & 1).flatten(1)[:, :v]
        out = torch.where(on != 0, out, torch.full_like(out, -math.inf))
    return out


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
    """The structures that describe the buffers to the library, the list of gradients and W in
    4 bits."""
    from macboost_amd import _core
    case, ctx = s["case"], _context()
    kind = case["kind"]
    if kind in ("embed", "embed_grad"):
        stride = case["dim"] + case["pad"]
        s["shape"] = _core.MbkEmbedShape(case["rows"], case["entries"], case["dim"],
                                         _CODES[case["type"]], stride, stride, case["scale"])
    elif kind == "clip":
        outs = s["outs"] or [None] * len(s["grads"])
        s["list"] = ctx.tensors([(_ptr(g), _ptr(o), g.shape[0], g.shape[1], g.stride(0),
                                  _core.F32 if g.dtype == torch.float32 else _core.BF16)
                                 for g, o in zip(s["grads"], outs)])
    elif kind == "scores":
        s["shape"] = _core.MbkFourbitShape(case["classes"], case["dim"], case["group"])
        w = s.pop("w")
        s["packed"] = torch.empty(_core.fourbit_bytes(s["shape"]), dtype=torch.uint8, device="cuda")
        ctx.call("mbk_fourbit_pack", ctypes.byref(s["shape"]), _CODES[case["type"]], _ptr(w),
                 w.stride(0), _ptr(s["packed"]))
    else:
        mask_stride = s["allowed"].stride(0) if case["mask"] == "row" else 0
        s["shape"] = _core.MbkAdjustShape(
            case["rows"], case["classes"], s["scores"].stride(0), s["out"].stride(0),
            case["history"], s["history"].stride(0), mask_stride, case["repetition"],
            case["presence"], case["frequency"])


def _own_run(s):
    ctx, case = _context(), s["case"]
    kind, ref = case["kind"], ctypes.byref
    if kind == "embed":
        ctx.call("mbk_embed", ref(s["shape"]), _ptr(s["table"]), _ptr(s["ids"]), _ptr(s["base"]),
                 _ptr(s["out"]))
    elif kind == "embed_grad":
        ctx.call("mbk_embed_grad", ref(s["shape"]), _ptr(s["ids"]), _ptr(s["dout"]),
                 _ptr(s["base"]), _ptr(s["out"]))
    elif kind == "clip":
        ctx.call("mbk_grad_clip", s["list"].ptr, s["max_norm"], _ptr(s["norm"]))
        return [s["norm"]] + list((s["buffers"] or {}).values())
    elif kind == "scores":
        ctx.call("mbk_fourbit_scores", ref(s["shape"]), case["rows"], _CODES[case["type"]],
                 _ptr(s["h"]), s["h"].stride(0), _ptr(s["packed"]), _ptr(s["bias"]),
                 _ptr(s["scores"]), s["scores"].stride(0))
        return s["scores"]
    else:
        ctx.call("mbk_adjust", ref(s["shape"]), _ptr(s["scores"]), _ptr(s["history"]),
                 _ptr(s["lengths"]), _ptr(s["bias"]), _ptr(s["allowed"]), _ptr(s["out"]))
    return s["out"]


def run(state):
    if own:
        return _own_run(state)
    return {"embed": _plain_embed, "embed_grad": _plain_embed_grad, "clip": _plain_clip,
            "scores": _plain_scores, "adjust": _plain_adjust}[state["case"]["kind"]](state)


# ---- the work -------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "clip":
        size = {"f32": 4, "bf16": 2}
        held = sum(r * c * size[t] for r, c, t in _tensor_shapes(case))
        elements = sum(r * c for r, c, _ in _tensor_shapes(case))
        if not case["ratio"]:
            return {"bytes": held + 4, "flops": 2 * elements}
        return {"bytes": 2 * held + 4, "flops": 3 * elements}
    n = case["rows"]
    if kind == "scores":
        v, d = case["classes"], case["dim"]
        groups = (d + case["group"] - 1) // case["group"]
        size = 4 if case["type"] == "f32" else 2
        moved = v * (d + 1) // 2 + 2 * v * groups + n * d * size + 4 * n * v
        return {"bytes": moved + (4 * v if case["bias"] else 0), "flops": 2 * n * v * d}
    if kind == "adjust":
        v = case["classes"]
        ids = n * case["history"] // (2 if case["ragged"] else 1)
        moved = 8 * n * v + 4 * ids + (4 * v if case["bias"] else 0) + \
            (4 * n if case["ragged"] else 0)
        if case["mask"] != "none":
            moved += 4 * ((v + 31) // 32) * (n if case["mask"] == "row" else 1)
        return {"bytes": moved, "flops": n * v * (1 if case["bias"] else 0) + 3 * ids}
    d, e = case["dim"], case["entries"]
    size = 4 if case["type"] == "f32" else 2
    kept = int(n * (1 - case["dropped"]))
    row = d * size
    if kind == "embed":
        # a vector that many rows take is read once
        moved = 4 * n + _distinct(case) * row + n * row * (2 if case["base"] else 1)
        return {"bytes": moved, "flops": kept * d * (2 if case["base"] else 1)}
    moved = 4 * n + kept * row + e * row * (2 if case["base"] else 1)
    return {"bytes": moved, "flops": kept * d + e * d * (2 if case["base"] else 1)}


def _distinct(case):
    """How many ids the kept rows hold, on average."""
    share = np.arange(1, case["entries"] + 1, dtype=np.float64) ** -case["skew"]
    share /= share.sum()
    kept = case["rows"] * (1 - case["dropped"])
    return int(np.sum(-np.expm1(kept * np.log1p(-np.minimum(share, 1 - 1e-12)))))


# ---- from the definitions, in 64 bits ---------------------------------------------

def _exact_embed(s):
    case = s["case"]
    width = case["dim"]
    padded = torch.zeros((case["entries"] + 1, width), dtype=torch.float64, device="cuda")
    padded[:-1] = s["table"]
    ids = torch.where(s["ids"] < 0, case["entries"], s["ids"]).long()
    out = torch.index_select(padded, 0, ids).mul_(_f32(case["scale"]))
    return out if s["base"] is None else out.add_(s["base"].double())


def _exact_embed_grad(s):
    case = s["case"]
    ids = s["ids"].cpu().numpy()
    order = np.argsort(ids, kind="stable")
    order = order[np.searchsorted(ids[order], 0):]
    out = np.zeros((case["entries"], case["dim"]))
    if order.size:
        used, first = np.unique(ids[order], return_index=True)
        rows = s["dout"].float().cpu().numpy()[order]
        out[used] = np.add.reduceat(rows, first, axis=0, dtype=np.float64)
    out = torch.from_numpy(out).cuda() * _f32(case["scale"])
    return out if s["base"] is None else out + s["base"].double()


def _exact_clip(s):
    squares = [torch.linalg.vector_norm(g.double()).item() for g in s["grads"]]
    norm = math.sqrt(math.fsum(x * x for x in squares))
    out = [torch.tensor([norm], dtype=torch.float64, device="cuda")]
    if math.isinf(s["max_norm"]):
        return out
    by = min(1.0, s["max_norm"] / norm) if norm else 1.0
    return out + [x.double() * by for x in s["held"].values()]


def _exact_scores(case, seed):
    gen = _generator(seed)
    n, d, v, dtype = case["rows"], case["dim"], case["classes"], _TYPES[case["type"]]
    h = _matrix(gen, n, d, case["pad"], dtype).double()
    w = _matrix(gen, v, d, 0, dtype, 2.0 / math.sqrt(d)).float()
    z = torch.zeros((n, v), dtype=torch.float64, device="cuda")
    for a in range(0, d, case["group"]):
        part = w[:, a:a + case["group"]]
        scale = (part.abs().max(1).values * _SEVENTH).bfloat16().float()[:, None]
        code = torch.round(part / scale).nan_to_num_(0.0, 0.0, 0.0).clamp_(-8, 7)
        z += torch.mm(h[:, a:a + case["group"]], (code.double() * scale.double()).t())
    if case["bias"]:
        bias = torch.empty(v, device="cuda").normal_(generator=gen).mul_(0.5)
        if case["masked"] > 0:
            bias[torch.rand(v, generator=gen, device="cuda") < case["masked"]] = -math.inf
        z += bias.double()
    return z


def _exact_adjust(s):
    case = s["case"]
    v = case["classes"]
    z = s["scores"].cpu().numpy().astype(np.float64)
    history = s["history"].cpu().numpy()
    lengths = None if s["lengths"] is None else s["lengths"].cpu().numpy()
    rep, presence, frequency = (_f32(case[k])
                                for k in ("repetition", "presence", "frequency"))
    for r in range(case["rows"]):
        seen = history[r] if lengths is None else history[r, :lengths[r]]
        ids, count = np.unique(seen, return_counts=True)
        was = z[r, ids]
        z[r, ids] = np.where(was > 0, was / rep, was * rep) - presence - frequency * count
    if s["bias"] is not None:
        z += s["bias"].cpu().numpy().astype(np.float64)
    if s["allowed"] is not None:
        words = s["allowed"].cpu().numpy().view(np.uint8)
        on = np.unpackbits(words, axis=1, bitorder="little")[:, :v].astype(bool)
        z[~np.broadcast_to(on, z.shape)] = -np.inf
    return torch.from_numpy(z).cuda()


def exact(case, seed):
    if case["kind"] == "scores":
        return _exact_scores(case, seed)
    s = prepare(case, seed)
    return {"embed": _exact_embed, "embed_grad": _exact_embed_grad, "clip": _exact_clip,
            "adjust": _exact_adjust}[case["kind"]](s)
