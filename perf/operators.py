"""What is measured of the operators on the parameter side of a training step: rows looked up in an embedding table, the
table's gradient, and the global norm of all gradients with their clipping.

Every case runs in two forms.  With `own` false the operators are written out in elementary torch operations, in 32 bits (64 for
long sums), rounded once at the end; with `own` true they are the framework's calls (`neuradar_amd.ops`).
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}


# ---------------------------------------------------------------------------------------------------------------- cases
def _rows(name, mode, n, rows, dim, dtype, index, order, scale=1.0, padding=-1):
    """A case on an embedding table [rows, dim] and n indices.  mode: "lookup" (the rows alone), "grad" (the table's gradient
    alone), "train" (both).  order: how the indices fall -- "uniform"; "skewed" (frequencies fall with the rank, like words in a
    text); "runs" (neighbours look up the same row, like the rays of one image).  padding: a row without a gradient, -1: none."""
    return {"name": name, "kind": "rows", "mode": mode, "n": n, "rows": rows, "dim": dim, "dtype": dtype, "index": index,
            "order": order, "scale": scale, "padding": padding}


def _clip(name, mode, layout, count, total, dtype, norm="2", ratio=0.5):
    """A case on a list of gradients.  mode: "norm" (the global norm alone), "clip" (norm and clipped gradients).  layout:
    "field" / "decoders" / "tables" (the shapes of this repository's own models) or "ragged" (`count` tensors of uneven sizes,
    `total` elements in all).  ratio: max_norm over the gradients' norm; at 1 and above nothing is clipped."""
    return {"name": name, "kind": "clip", "mode": mode, "layout": layout, "count": count, "total": total, "dtype": dtype,
            "norm": norm, "ratio": ratio}


def listed():
    return [
        # one 32 x 32 camera patch looks up its appearance rows (3 sensors x 20 s at 1 Hz, 16 wide): a latency
        _rows("lookup_patch", "lookup", 1024, 60, 16, "float32", "int64", "runs"),
        # odd everything: a row of 66 bytes starts at any 2-byte address
        _rows("lookup_odd", "lookup", 50021, 10007, 33, "float16", "int32", "uniform", 5.744562646538029),
        # token rows of a long batch, scaled by sqrt(dim): writes half a gigabyte
        _rows("lookup_tokens", "lookup", 262144, 131072, 1024, "bfloat16", "int64", "skewed", 32.0),
        # a step of 16 384 rays through the appearance table: 273 rays to a row, rows and gradient
        _rows("train_appearance", "train", 16384, 60, 16, "float32", "int64", "runs"),
        # the rays of the reference's whole batch (40 960 camera, 16 384 lidar, 16 radar scans of 3 531) and a row for each image
        _rows("grad_images", "grad", 113840, 1999, 32, "float32", "int64", "runs"),
        # few indices into a table of 2^22 rows: the gradient is nearly all zeros, and it is written whole
        _rows("grad_sparse", "grad", 8192, 1 << 22, 8, "float32", "int32", "uniform"),
        # a language model's token table in training: skewed, one row is padding
        _rows("train_tokens", "train", 131072, 131072, 512, "bfloat16", "int64", "skewed", 22.627416997969522, 0),
        # seven classes over a long batch, odd width: runs of 14 000 equal indices
        _rows("grad_classes", "grad", 100003, 7, 257, "float32", "int32", "uniform"),
        # gradients of the field's networks: two dozen small tensors, a latency
        _clip("norm_field", "norm", "field", 0, 0, "float32"),
        # the camera and radar decoders' gradients: 7 x 7 convolutions, a transformer layer, biases and norms
        _clip("clip_decoders", "clip", "decoders", 0, 0, "float32"),
        # a long ragged list in 16 bits, as a transformer of many layers leaves it
        _clip("clip_ragged", "clip", "ragged", 288, 1 << 26, "bfloat16"),
        # every table of the default model and its small parameters, 153 million elements in all: the largest
        _clip("clip_tables", "clip", "tables", 0, 0, "float32"),
    ]


def _log_int(rng, low, high):
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return min(max(v, low), high)


def draw(rng):
    if rng.random() < 0.65:
        dtype = rng.choice(["float32", "bfloat16", "float16"])
        while True:
            n, rows, dim = _log_int(rng, 1, 1 << 18), _log_int(rng, 1, 1 << 22), _log_int(rng, 1, 1024)
            if rng.random() < 0.5:  # half of the widths are whole 16-byte groups, half are whatever comes
                dim = max(8, dim // 8 * 8)
            if n * dim <= 1 << 27 and rows * dim <= 1 << 26:
                break
        mode = rng.choice(["lookup", "grad", "train"])
        case = _rows("", mode, n, rows, dim, dtype, rng.choice(["int32", "int64"]), rng.choice(["uniform", "skewed", "runs"]),
                     rng.choice([1.0, 0.5, math.sqrt(dim)]), rng.choice([-1, rng.randrange(rows)]))
    else:
        count = _log_int(rng, 1, 320)
        total = max(count, _log_int(rng, 64, 1 << 27))
        case = _clip("", rng.choice(["norm", "clip", "clip"]), "ragged", count, total, rng.choice(["float32", "bfloat16", "float16"]),
                     rng.choice(["2", "2", "1", "inf"]), rng.choice([0.01, 0.5, 0.999, 2.0]))
    del case["name"]
    return case


# --------------------------------------------------------------------------------------------------------------- inputs
def _sizes(case):
    """Elements of each tensor of a clip case."""
    if case["layout"] == "field":  # geometry and feature networks (weights and biases), beta, the proposal heads, the lidar network
        mlp = [32 * 32, 32, 32 * 33, 33, 48 * 32, 32, 32 * 32, 32, 32 * 32, 32, 1, 6, 6]
        return mlp + [48 * 32, 32, 32 * 32, 32, 32 * 2, 2, 60 * 16]
    if case["layout"] == "decoders":  # 48 wide: 4 residual blocks of two convolutions, up-sampling, a 48 / 64 encoder layer, 4 heads
        block = [32 * 32 * 49, 32, 32, 32] * 2
        encoder = [144 * 48, 144, 48 * 48, 48, 64 * 48, 64, 48 * 64, 48] + [48] * 6
        return [48 * 32, 32] + block * 4 + [32 * 32 * 9, 32, 32 * 3, 3] + encoder + [48 * 32, 32, 32 * 32, 32, 32 * 3, 3] * 4
    if case["layout"] == "tables":  # main table, its actors' share, two proposal tables, small parameters in one buffer
        return [(1 << 22) * 8 * 4, (1 << 20) * 6, (1 << 20) * 6, 12 * (1 << 17) * 4, 250007]
    rng = np.random.default_rng(case["count"] * 7919 + case["total"])  # (the sizes are the case's, the values the seed's)
    share = rng.lognormal(0.0, 1.5, case["count"])
    sizes = np.maximum(1, np.floor(share / share.sum() * case["total"])).astype(np.int64)
    return [int(s) for s in sizes]


def _indices(case, gen):
    n, rows = case["n"], case["rows"]
    if case["order"] == "uniform":
        idx = torch.randint(0, rows, (n,), device="cuda", generator=gen)
    elif case["order"] == "skewed":  # rank r with a frequency like 1 / r; the ranks lie anywhere in the table
        u = torch.rand(n, device="cuda", generator=gen, dtype=torch.float64)
        rank = (torch.exp(u * math.log(rows + 1.0)) - 1.0).long().clamp_(0, rows - 1)
        idx = (rank * 2654435761 + 12345) % rows
    else:  # runs of up to 256 equal ones
        length = max(1, min(256, n // 4))
        heads = torch.randint(0, rows, ((n + length - 1) // length,), device="cuda", generator=gen)
        idx = heads.repeat_interleave(length)[:n]
    return idx.to(torch.int32 if case["index"] == "int32" else torch.int64)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "rows":
        state = {"case": case, "idx": _indices(case, gen), "scale": case["scale"],
                 "padding": None if case["padding"] < 0 else case["padding"]}
        if case["mode"] != "grad":
            state["table"] = (torch.randn(case["rows"], case["dim"], device="cuda", generator=gen) * 0.5).to(dtype)
        if case["mode"] != "lookup":
            state["grad"] = torch.randn(case["n"], case["dim"], device="cuda", generator=gen).mul_(1.0 / 64).to(dtype)
        return state
    grads, sizes = [], _sizes(case)
    spread = torch.rand(len(sizes), generator=torch.Generator().manual_seed(seed)).mul_(3.0).sub_(3.0)  # 1e-3 ... 1
    for size, power in zip(sizes, spread.tolist()):
        grads.append(torch.randn(size, device="cuda", generator=gen).mul_(10.0 ** power).to(dtype))
    norm = float(_norm64(grads, case["norm"]))
    # a program keeps the bucket that its clipped gradients go to; each has a place in it that starts on 16 bytes
    bucket = torch.zeros(sum(_places(case)) if case["mode"] == "clip" else 0, device="cuda", dtype=dtype)
    out = [b[:g.numel()] for b, g in zip(bucket.split(_places(case)), grads)] if case["mode"] == "clip" else None
    return {"case": case, "grads": grads, "max_norm": norm * case["ratio"], "out": out, "bucket": bucket}


def _places(case):
    group = 16 // BYTES[case["dtype"]]
    return [(s + group - 1) // group * group for s in _sizes(case)]


def _norm64(grads, norm):
    if norm == "inf":
        return torch.stack([g.abs().max().double() for g in grads]).max()
    if norm == "1":
        return torch.stack([g.abs().sum(dtype=torch.float64) for g in grads]).sum()
    return torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()


# ------------------------------------------------------------------------------------------------------------- one pass
def _lookup(table, idx, scale):
    return (table[idx].float() * scale).to(table.dtype)


def _table_gradient(grad, idx, rows, scale, padding):
    # (runs of thousands of equal indices are long sums)
    wide = torch.float64 if grad.shape[0] >= 4096 * rows else torch.float32
    values = grad.to(wide)
    if padding is not None:
        values = torch.where((idx != padding)[:, None], values, torch.zeros((), device=values.device, dtype=wide))
    total = torch.zeros(rows, grad.shape[1], device=grad.device, dtype=wide).index_add_(0, idx, values)
    return (total * scale).to(grad.dtype)


def _global_norm(grads, norm):
    if norm == "inf":
        return torch.stack([g.float().abs().max() for g in grads]).max()
    if norm == "1":
        return torch.stack([g.float().abs().sum() for g in grads]).sum()
    return torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()


def run(state):
    case = state["case"]
    if own:
        from neuradar_amd import ops
    if case["kind"] == "rows":
        outputs = {}
        if case["mode"] != "grad":
            lookup = ops.embedding if own else _lookup
            outputs["rows"] = lookup(state["table"], state["idx"], state["scale"])
        if case["mode"] != "lookup":
            gradient = ops.embedding_grad if own else _table_gradient
            outputs["grad"] = gradient(state["grad"], state["idx"], case["rows"], state["scale"], state["padding"])
        return outputs
    norm_type = float(case["norm"])
    if case["mode"] == "norm":
        return {"norm": ops.grad_norm(state["grads"], norm_type) if own else _global_norm(state["grads"], case["norm"])}
    if own:
        norm = ops.clip_grads(state["grads"], state["max_norm"], norm_type, out=state["out"])
        return {"norm": norm, "grads": state["bucket"]}
    norm = _global_norm(state["grads"], case["norm"])
    factor = torch.clamp(state["max_norm"] / (norm + 1e-6), max=1.0)
    for place, g in zip(state["out"], state["grads"]):
        place.copy_(g.float() * factor)
    return {"norm": norm, "grads": state["bucket"]}


def work(case):
    size = BYTES[case["dtype"]]
    if case["kind"] == "rows":
        n, rows, dim = case["n"], case["rows"], case["dim"]
        bytes_, flops = n * (4 if case["index"] == "int32" else 8), 0
        touched = min(n, rows)  # (a row that is looked up often is read once)
        if case["mode"] != "grad":
            bytes_ += (touched + n) * dim * size
            flops += n * dim
        if case["mode"] != "lookup":
            bytes_ += (n + rows) * dim * size
            flops += n * dim + touched * dim
        return {"bytes": bytes_, "flops": flops}
    total = sum(_sizes(case))
    if case["mode"] == "norm":
        return {"bytes": total * size + 4, "flops": 2 * total}
    return {"bytes": 2 * total * size + 4, "flops": 3 * total}


# ------------------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "rows":
        idx = state["idx"].long().cpu().numpy()
        outputs = {}
        if case["mode"] != "grad":
            outputs["rows"] = np.take(state["table"].double().cpu().numpy(), idx, axis=0) * case["scale"]
        if case["mode"] != "lookup":
            # equal indices brought together, each run summed by itself
            grad = state["grad"].double().cpu().numpy()
            order = np.argsort(idx, kind="stable")
            if case["padding"] >= 0:
                order = order[idx[order] != case["padding"]]
            total = np.zeros((case["rows"], case["dim"]))
            if order.size:
                first = np.flatnonzero(np.r_[True, idx[order][1:] != idx[order][:-1]])
                total[idx[order][first]] = np.add.reduceat(grad[order], first, axis=0) * case["scale"]
            outputs["grad"] = total
        return outputs
    norm = float(_norm64(state["grads"], case["norm"]))
    if case["mode"] == "norm":
        return {"norm": np.float64(norm)}
    factor = min(1.0, state["max_norm"] / (norm + 1e-6))
    whole = []
    for g, place in zip(state["grads"], _places(case)):
        whole += [g.double() * factor, torch.zeros(place - g.numel(), device="cuda", dtype=torch.float64)]
    return {"norm": np.float64(norm), "grads": torch.cat(whole)}
