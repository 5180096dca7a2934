"""Workloads of the row operators: LayerNorm and the embedding lookup, forward and backward.

They are the step between the tensors the image operators of this library produce (and the token ids that come with them)
and the first activations of the model they feed: normalising image patches, channels or whole images by their own
statistics, looking up rows of a table by index (tokens, positions, class labels, palette colours), and the gradients of
both. Every workload has a plain form made of elementary torch operations in 32 bits, and the library's own call.
"""
from __future__ import annotations

import importlib.util
import math
import os
import sys

import torch

own = False

_DT = {"u8": torch.uint8, "f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "i32": torch.int32,
       "i64": torch.int64}
_SIZE = {"u8": 1, "f16": 2, "bf16": 2, "f32": 4, "i32": 4, "i64": 8, None: 0}
_EPS = 1e-5
# elements of the largest listed tensor: 256 images of 224 x 224 x 3, 196 patches of 16 x 16 x 3 each
_MOST = 256 * 224 * 224 * 3

_package = None


def _pkg():
    global _package
    if _package is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        name = "cvcuda_b200"
        if name not in sys.modules:
            folder = os.path.join(root, "cv-cuda_b200")
            spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"),
                                                          submodule_search_locations=[folder])
            sys.modules[name] = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(sys.modules[name])
        _package = sys.modules[name]
    return _package


def _ln(name, rows, cols, src, dst, wtype, **more):
    return {"name": name, "op": "layernorm", "rows": rows, "cols": cols, "src": src, "dst": dst, "weight": wtype, "stats": False,
            "image": False, **more}


def _ln_bwd(name, rows, cols, src, grad, wtype, **more):
    return {"name": name, "op": "layernorm_backward", "rows": rows, "cols": cols, "src": src, "grad": grad, "weight": wtype,
            "dsrc": True, **more}


def _emb(name, count, rows, cols, ids, table, dst, scale, **more):
    return {"name": name, "op": "embedding", "count": count, "rows": rows, "cols": cols, "ids": ids, "table": table, "dst": dst,
            "scale": scale, "outside": False, **more}


def _emb_bwd(name, count, rows, cols, ids, grad, dst, scale, **more):
    return {"name": name, "op": "embedding_backward", "count": count, "rows": rows, "cols": cols, "ids": ids, "grad": grad,
            "dst": dst, "scale": scale, "padding": -1, "outside": False, "zipf": 1.0, **more}


def listed():
    return [
        # one token of a sequence being generated: a single row, where only latency counts
        _ln("ln_one_token", 1, 4096, "bf16", "bf16", "bf16"),
        # the patches of a batch of pre-processed images: 256 images of 224 x 224, 196 patches of 16 x 16 x 3 each
        _ln("ln_patches", 50176, 768, "f16", "f16", "f32"),
        # 14 x 14 x 3 patches of 64 float32 images: a row length that is no multiple of eight; statistics kept for training
        _ln("ln_patches_14", 16384, 588, "f32", "bf16", "f32", stats=True),
        # per-image standardisation of a uint8 batch: a whole 224 x 224 x 3 image is one row, no weights
        _ln("ln_images_u8", 256, 224 * 224 * 3, "u8", "f32", None, image=True),
        # training step over the patches of ln_patches: gradients of input, weight and bias
        _ln_bwd("ln_bwd_patches", 50176, 768, "bf16", "bf16", "f32"),
        # ragged in every direction: odd row length, odd number of rows
        _ln_bwd("ln_bwd_odd", 5003, 2051, "f16", "f16", "f16"),
        # a few class tokens: latency again
        _ln_bwd("ln_bwd_few", 17, 1000, "f32", "f32", "f32"),
        # the tokens of four sequences being generated
        _emb("emb_four_tokens", 4, 32000, 4096, "i64", "bf16", "bf16", 64.0),
        # a batch of prompts: 32 sequences of 2048 tokens, the table scaled by the square root of its width
        _emb("emb_prompts", 65536, 50000, 1024, "i32", "bf16", "bf16", 32.0),
        # eight 1080p label maps to colours: uint8 indices, a palette of three channels
        _emb("emb_palette", 8 * 1080 * 1920, 256, 3, "u8", "f32", "f16", 1.0 / 255.0),
        # training step: 16384 tokens of natural frequency, padding left out, float32 gradient of the whole table
        _emb_bwd("emb_bwd_tokens", 16384, 32000, 1024, "i64", "bf16", "f32", 32.0, padding=0),
        # class labels: few table rows, each used many times, odd sizes
        _emb_bwd("emb_bwd_labels", 5003, 1000, 333, "i32", "f32", "f32", 1.0, zipf=0.0),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["layernorm", "layernorm", "layernorm_backward", "embedding", "embedding_backward"])
    if op == "layernorm":
        src = rng.choice(["u8", "f16", "bf16", "f32"])
        dst = rng.choice(["f16", "bf16", "f32"])
        if rng.random() < 0.25:  # whole images as rows
            cols = _log_int(rng, 28, 448) * _log_int(rng, 28, 448) * rng.choice([1, 3, 4])
            return {"op": op, "rows": _log_int(rng, 1, max(1, _MOST // cols)), "cols": cols, "src": src, "dst": dst,
                    "weight": None, "stats": rng.random() < 0.5, "image": True}
        cols = _log_int(rng, 8, 16384)
        if rng.random() < 0.5:
            cols = max(8, cols // 8 * 8)
        return {"op": op, "rows": _log_int(rng, 1, max(1, min(1 << 20, _MOST // cols))), "cols": cols, "src": src, "dst": dst,
                "weight": rng.choice([None, "f16", "bf16", "f32"]), "stats": rng.random() < 0.5, "image": False}
    if op == "layernorm_backward":
        cols = _log_int(rng, 8, 16384)
        if rng.random() < 0.5:
            cols = max(8, cols // 8 * 8)
        src = rng.choice(["u8", "f16", "bf16", "f32"])
        return {"op": op, "rows": _log_int(rng, 1, max(1, min(1 << 19, _MOST // cols))), "cols": cols, "src": src,
                "grad": rng.choice(["f16", "bf16", "f32"]) if src == "u8" else src,
                "weight": rng.choice([None, "f32", "bf16"]), "dsrc": src != "u8"}
    ids = rng.choice(["u8", "i32", "i64"])
    rows = 256 if ids == "u8" else _log_int(rng, 10, 65536)
    cols = _log_int(rng, 3 if op == "embedding" else 16, 4096)
    if rng.random() < 0.5:
        cols = max(8, cols // 8 * 8)
    rows = max(1, min(rows, 50000 * 1024 // cols))
    count = _log_int(rng, 1, max(1, min(65536, _MOST // cols)))
    outside = ids != "u8" and rng.random() < 0.3
    scale = rng.choice([1.0, math.sqrt(cols), 0.125])
    kind = rng.choice(["f16", "bf16", "f32"])
    if op == "embedding":
        return {"op": op, "count": count, "rows": rows, "cols": cols, "ids": ids, "table": kind,
                "dst": rng.choice([kind, "f32"]), "scale": scale, "outside": outside}
    return {"op": op, "count": count, "rows": rows, "cols": cols, "ids": ids, "grad": kind, "dst": rng.choice(["f32", kind]),
            "scale": scale, "padding": rng.choice([-1, 0]), "outside": outside, "zipf": rng.choice([0.0, 1.0])}


def _values(gen, shape, kind):
    if kind == "u8":
        return torch.randint(0, 256, shape, generator=gen, device="cuda", dtype=torch.uint8)
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(_DT[kind])


def _indices(gen, case):
    n, rows = case["count"], case["rows"]
    if case.get("zipf", 1.0) > 0:  # frequencies that fall as 1 / rank, ranks spread over the table
        u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
        ids = (torch.exp(u * math.log(rows + 1.0)) - 1.0).long().clamp_(0, rows - 1)
        ids = torch.where(ids == 0, ids, (ids * 7919) % rows)
    else:
        ids = torch.randint(0, rows, (n,), generator=gen, device="cuda")
    if case["outside"]:  # a table that holds a part of the indices: the others belong to another part
        ids = torch.where(torch.rand(n, generator=gen, device="cuda") < 0.5, ids, ids + rows)
    if case["ids"] == "u8":
        ids = ids % 256
    return ids.to(_DT[case["ids"]])


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = {"case": case}
    cols = case["cols"]
    if case["op"] in ("layernorm", "layernorm_backward"):
        x = _values(gen, (case["rows"], cols), case["src"])
        if case["src"] != "u8":
            # rows with offsets and sizes of their own, as activations have
            spread = 0.5 + torch.rand((case["rows"], 1), generator=gen, device="cuda")
            offset = torch.randn((case["rows"], 1), generator=gen, device="cuda")
            x = (x.float() * spread + offset).to(_DT[case["src"]])
        state["src"] = x
        state["weight"] = state["bias"] = None
        if case["weight"] is not None:
            state["weight"] = (1.0 + 0.2 * torch.randn(cols, generator=gen, device="cuda")).to(_DT[case["weight"]])
            state["bias"] = (0.2 * torch.randn(cols, generator=gen, device="cuda")).to(_DT[case["weight"]])
        if case["op"] == "layernorm_backward":
            state["grad"] = _values(gen, (case["rows"], cols), case["grad"])
            # what the forward pass left behind
            mean = torch.empty(case["rows"], device="cuda")
            rstd = torch.empty(case["rows"], device="cuda")
            step = max(1, (1 << 24) // cols)
            for i in range(0, case["rows"], step):
                part = x[i:i + step].double()
                m = part.mean(1, keepdim=True)
                mean[i:i + step] = m[:, 0].float()
                rstd[i:i + step] = (1.0 / torch.sqrt(((part - m) ** 2).mean(1) + _EPS)).float()
            state["mean"], state["rstd"] = mean, rstd
        return state
    state["ids"] = _indices(gen, case)
    if case["op"] == "embedding":
        state["table"] = _values(gen, (case["rows"], cols), case["table"])
        if case["cols"] <= 4:
            state["table"] = (state["table"].float().abs() * 80.0).clamp_(0, 255).to(_DT[case["table"]])
    else:
        state["grad"] = _values(gen, (case["count"], cols), case["grad"])
    return state


def _run_own(state):
    case, pkg = state["case"], _pkg()
    if case["op"] == "layernorm":
        return pkg.layernorm(state["src"], state["weight"], state["bias"], _EPS, data_type=_DT[case["dst"]], stats=case["stats"])
    if case["op"] == "layernorm_backward":
        affine = case["weight"] is not None
        return [g for g in pkg.layernorm_backward(state["grad"], state["src"], state["mean"], state["rstd"], state["weight"],
                                                  src_grad=case["dsrc"], weight_grad=affine or not case["dsrc"],
                                                  bias_grad=affine or not case["dsrc"]) if g is not None]
    if case["op"] == "embedding":
        return pkg.embedding(state["ids"], state["table"], case["scale"], data_type=_DT[case["dst"]])
    return pkg.embedding_backward(state["grad"], state["ids"], case["rows"], case["scale"],
                                  padding_index=None if case["padding"] < 0 else case["padding"], data_type=_DT[case["dst"]])


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["op"] == "layernorm":
        x = state["src"].float()
        mean = x.mean(1, keepdim=True)
        x = x - mean
        rstd = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + _EPS)
        y = x * rstd
        if state["weight"] is not None:
            y = y * state["weight"].float() + state["bias"].float()
        y = y.to(_DT[case["dst"]])
        return (y, mean[:, 0], rstd[:, 0]) if case["stats"] else y
    if case["op"] == "layernorm_backward":
        g = state["grad"].float()
        xhat = (state["src"].float() - state["mean"][:, None]) * state["rstd"][:, None]
        out = []
        if case["dsrc"]:
            gw = g if state["weight"] is None else g * state["weight"].float()
            c1 = gw.mean(1, keepdim=True)
            c2 = (gw * xhat).mean(1, keepdim=True)
            out.append(((gw - c1 - xhat * c2) * state["rstd"][:, None]).to(_DT[case["src"]]))
        if state["weight"] is not None or not case["dsrc"]:
            kind = torch.float32 if state["weight"] is None else state["weight"].dtype
            out += [(g * xhat).sum(0).to(kind), g.sum(0).to(kind)]
        return out
    ids = state["ids"].long()
    if case["op"] == "embedding":
        table = state["table"]
        if not case["outside"]:
            return (table[ids].float() * case["scale"]).to(_DT[case["dst"]])
        here = (ids >= 0) & (ids < case["rows"])
        y = table[torch.where(here, ids, 0)].float() * case["scale"]
        return torch.where(here[:, None], y, 0.0).to(_DT[case["dst"]])
    g = state["grad"].float() * case["scale"]
    if case["outside"] or case["padding"] >= 0:
        left_out = (ids < 0) | (ids >= case["rows"])
        if case["padding"] >= 0:
            left_out = left_out | (ids == case["padding"])
        ids = torch.where(left_out, 0, ids)
        g = torch.where(left_out[:, None], 0.0, g)
    out = torch.zeros((case["rows"], case["cols"]), device="cuda")
    out.index_add_(0, ids, g)
    return out.to(_DT[case["dst"]])


def work(case):
    cols = case["cols"]
    if case["op"] == "layernorm":
        n = case["rows"] * cols
        return {"bytes": n * (_SIZE[case["src"]] + _SIZE[case["dst"]]) + 2 * cols * _SIZE[case["weight"]]
                + (8 * case["rows"] if case["stats"] else 0), "flops": 8 * n}
    if case["op"] == "layernorm_backward":
        n = case["rows"] * cols
        w = _SIZE[case["weight"]]
        params = cols * (3 * w if w else (0 if case["dsrc"] else 8))
        return {"bytes": n * (_SIZE[case["src"]] + _SIZE[case["grad"]] + (_SIZE[case["src"]] if case["dsrc"] else 0)) + 8 * case["rows"]
                + params, "flops": 14 * n}
    n = case["count"] * cols
    if case["op"] == "embedding":
        # table rows that are read at all: expected number of different indices, at most the table
        used = min(case["count"], case["rows"])
        if case["count"] > 16:
            used = min(used, _different(case))
        return {"bytes": used * cols * _SIZE[case["table"]] + n * _SIZE[case["dst"]] + case["count"] * _SIZE[case["ids"]], "flops": n}
    return {"bytes": n * _SIZE[case["grad"]] + case["count"] * _SIZE[case["ids"]] + case["rows"] * cols * _SIZE[case["dst"]],
            "flops": 2 * n}


def _different(case):
    """Expected number of different table rows among the indices, whose rank has density 1 / ((1 + r) log(rows + 1))."""
    total, r, rows, n = 0.0, 0, case["rows"], case["count"] * (0.5 if case["outside"] else 1.0)
    while r < rows:
        step = max(1, r // 64)
        p = math.log((r + 1.0 + step) / (r + 1.0)) / math.log(rows + 1.0) / step
        total += step * (1.0 - math.exp(n * math.log1p(-min(p, 1.0 - 1e-12))))
        r += step
    return int(min(rows, total)) + 1


def exact(case, seed):
    """The definitions, in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "layernorm":
        x = s["src"].double()
        n = x.shape[1]
        mu = x.sum(1) / n
        var = torch.stack([((r - m) ** 2).sum() / n for r, m in zip(x, mu)]) if x.shape[0] <= 64 else (x - mu[:, None]).pow(2).sum(1) / n
        rs = (var + _EPS).pow(-0.5)
        y = (x - mu[:, None]) * rs[:, None]
        if s["weight"] is not None:
            y = s["weight"].double()[None, :] * y + s["bias"].double()[None, :]
        return (y, mu, rs) if case["stats"] else y
    if case["op"] == "layernorm_backward":
        # y_j = w_j h_j + b_j, h = (x - mu) rs: dh = w dy; dx_k = rs (dh_k - sum(dh) / n - h_k sum(dh h) / n)
        x, dy, rs = s["src"].double(), s["grad"].double(), s["rstd"].double()[:, None]
        h = (x - s["mean"].double()[:, None]) * rs
        out = []
        if case["dsrc"]:
            dh = dy if s["weight"] is None else dy * s["weight"].double()[None, :]
            n = x.shape[1]
            out.append(rs / n * (n * dh - dh.sum(1, keepdim=True) - h * (dh * h).sum(1, keepdim=True)))
        if s["weight"] is not None or not case["dsrc"]:
            out += [torch.einsum("rc,rc->c", dy, h), dy.sum(0)]
        return out
    ids = s["ids"].long()
    inside = (ids >= 0) & (ids < case["rows"])
    if case["op"] == "embedding":
        y = torch.zeros((case["count"], case["cols"]), dtype=torch.float64, device="cuda")
        y[inside] = s["table"].double()[ids[inside]] * case["scale"]
        return y
    if case["padding"] >= 0:
        inside &= ids != case["padding"]
    out = torch.zeros((case["rows"], case["cols"]), dtype=torch.float64, device="cuda")
    return out.index_put_((ids[inside],), s["grad"].double()[inside] * case["scale"], accumulate=True)
