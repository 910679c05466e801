"""Products with block-sparse 8-bit matrices, and the 8-bit rows that go with them: serving one to thirty-two rows, products of
many rows, activations kept in 8 bits between the passes of a training step, both gradients, and new values of the matrix.

A matrix has n_rows x n_cols entries, of which 128 x 128 blocks are stored (the blocks that pruning has left); a block holds e4m3
values and one scale. Rows (activations) are e4m3 with one scale for each 128 columns. A scale is the smallest power of two for which
no finite magnitude of its block is above 448 (2^-126 at least), so that what 8 bits stand for is exact in 16.

    single      y = A x for one row or a few, given in 16 or 32 bits: the decoding step
    product     y = A x for many rows: the forward pass of a layer
    checkpoint  rows to 8 bits and back: an activation kept for the backward pass
    backward    from the checkpoint of x and from dy: dx = A^T dy (dy in 8 bits, too) and dA = dy x^T for the stored blocks
    update      new values of the stored blocks, from 32 bits
    step        update, forward pass and backward pass of one layer
"""
from __future__ import annotations

import torch

own = False

BLOCK = 128
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one token of one sequence through a pruned projection: the smallest call, all of it latency
        {"name": "single-1x1024x1024", "kind": "single", "tokens": 1, "rows": 1024, "cols": 1024, "density": 0.5, "dtype": "bf16"},
        # one token through a wide layer of which nothing is pruned: as fast as the matrix can be read
        {"name": "single-1x8192x8192", "kind": "single", "tokens": 1, "rows": 8192, "cols": 8192, "density": 1.0, "dtype": "bf16"},
        # a decoding batch, the last of the sequences ragged, a matrix that ends inside blocks
        {"name": "single-19x4001x2047", "kind": "single", "tokens": 19, "rows": 4001, "cols": 2047, "density": 0.6, "dtype": "f32"},
        # a batch of prompts through a layer of which a quarter is left
        {"name": "product-2048x4096x4096", "kind": "product", "tokens": 2048, "rows": 4096, "cols": 4096, "density": 0.25, "dtype": "bf16"},
        # a few hundred tokens: too many for the decoding kernel, too few to fill the chip by themselves
        {"name": "product-333x1801x1603", "kind": "product", "tokens": 333, "rows": 1801, "cols": 1603, "density": 0.7, "dtype": "f16"},
        # the largest product: bounded by the tensor cores
        {"name": "product-8192x8192x8192", "kind": "product", "tokens": 8192, "rows": 8192, "cols": 8192, "density": 0.5, "dtype": "bf16"},
        # an activation of a training step, kept in 8 bits and read back
        {"name": "checkpoint-8192x4096", "kind": "checkpoint", "tokens": 8192, "cols": 4096, "pad": 0, "dtype": "bf16"},
        # columns of a wider activation, at an odd distance
        {"name": "checkpoint-1603x1801", "kind": "checkpoint", "tokens": 1603, "cols": 1801, "pad": 250, "dtype": "f32"},
        # the backward pass of a pruned layer
        {"name": "backward-4096x4096x4096", "kind": "backward", "tokens": 4096, "rows": 4096, "cols": 4096, "density": 0.25, "dtype": "bf16"},
        # the same for a layer and a batch that fill no block, in half precision
        {"name": "backward-1001x1000x1201", "kind": "backward", "tokens": 1001, "rows": 1000, "cols": 1201, "density": 0.5, "dtype": "f16"},
        # the optimiser has stepped: new values of a whole layer
        {"name": "update-8192x4096", "kind": "update", "rows": 8192, "cols": 4096, "density": 0.5},
        # everything a layer does in one step of training
        {"name": "step-8192x8192x4096", "kind": "step", "tokens": 8192, "rows": 8192, "cols": 4096, "density": 0.25, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["single", "single", "product", "product", "checkpoint", "backward", "backward", "update", "step"])
    density = round(0.05 * 20.0 ** rng.random(), 3)
    if kind == "single":
        return {"kind": kind, "tokens": _log(rng, 1, 32), "rows": _log(rng, 128, 8192), "cols": _log(rng, 128, 8192), "density": density,
                "dtype": rng.choice(["bf16", "f16", "f32"])}
    if kind == "product":
        return {"kind": kind, "tokens": _log(rng, 33, 8192), "rows": _log(rng, 128, 8192), "cols": _log(rng, 128, 8192), "density": density,
                "dtype": rng.choice(["bf16", "f16", "f32"])}
    if kind == "checkpoint":
        return {"kind": kind, "tokens": _log(rng, 1, 8192), "cols": _log(rng, 100, 8192), "pad": rng.choice([0, 0, 8, rng.randint(1, 200)]),
                "dtype": rng.choice(["bf16", "f16", "f32"])}
    if kind == "update":
        return {"kind": kind, "rows": _log(rng, 128, 8192), "cols": _log(rng, 128, 4096), "density": density}
    return {"kind": kind, "tokens": _log(rng, 33, 8192), "rows": _log(rng, 128, 8192), "cols": _log(rng, 128, 4096), "density": density,
            "dtype": rng.choice(["bf16", "f16"])}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _blocks(n):
    return -(-n // BLOCK)


def _pattern(case, seed):
    """Which blocks are stored, as many as the case's density says; a layer of several block rows has lost one of them entirely."""
    g = torch.Generator()
    g.manual_seed(int(seed))
    score = torch.rand(_blocks(case["rows"]), _blocks(case["cols"]), generator=g)
    n, full = max(1, round(case["density"] * score.numel())), score.numel()
    if case["density"] < 1.0 and score.shape[0] >= 4:
        score[int(torch.randint(0, score.shape[0], (1,), generator=g))] = 2.0
        full -= score.shape[1]
    kept = torch.zeros(score.numel(), dtype=torch.bool)
    kept[score.reshape(-1).argsort()[: min(n, full)]] = True
    return kept.reshape(score.shape)


def _activations(g, tokens, width, dtype):
    """A few columns are much larger than the others, as in trained models; the last rows of a batch may be padding."""
    x = torch.randn(tokens, width, generator=g, device="cuda") * torch.exp(1.5 * torch.randn(width, generator=g, device="cuda")).clamp(max=60.0)
    if tokens > 64:
        x[-(tokens // 50):] = 0.0
    return x.to(dtype)


def _inside(n):
    """For each row (or column) of the blocks: whether the matrix has it."""
    return (torch.arange(_blocks(n) * BLOCK, device="cuda") < n).reshape(-1, BLOCK)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    kind = case["kind"]
    s = {"kind": kind}
    if "dtype" in case:
        s["dtype"] = case["dtype"]
    if "rows" in case:
        kept = _pattern(case, seed)
        at = kept.nonzero()
        n = at.shape[0]
        w = torch.randn(n, BLOCK, BLOCK, generator=g, device="cuda") * case["cols"] ** -0.5 * torch.exp(0.5 * torch.randn(n, 1, 1, generator=g, device="cuda"))
        w *= _inside(case["rows"])[at[:, 0].cuda()][:, :, None] & _inside(case["cols"])[at[:, 1].cuda()][:, None, :]
        s.update(rows=case["rows"], cols=case["cols"], block_row=at[:, 0].cuda(), block_col=at[:, 1].cuda())
        s["master"] = w  # 32 bits, what the optimiser keeps
        if kind not in ("update", "step"):
            s["values"] = _eight_bits(w.reshape(n, -1), BLOCK * BLOCK).reshape(n, BLOCK, BLOCK)  # what the stored matrix stands for
    if "tokens" in case:
        dtype, pad = TYPES[case["dtype"]], case.get("pad", 0)
        s["x"] = _activations(g, case["tokens"], case["cols"] + pad, dtype)[:, : case["cols"]]
        if kind in ("backward", "step"):
            s["dy"] = (1e-2 * torch.randn(case["tokens"], case["rows"], generator=g, device="cuda") * torch.exp(torch.randn(case["tokens"], 1, generator=g, device="cuda"))).to(dtype)
        if kind == "backward":
            s["x"] = _eight_bits(s["x"], BLOCK).to(dtype)  # what the checkpoint of the forward pass stands for
    if own:
        _handles(s, case)
    return s


def _handles(s, case):
    """What a program keeps between its calls: the matrix in the library's form, the checkpoints' room, and its own results' buffers."""
    import numpy as np

    from alphasparse_b200 import capi
    from alphasparse_b200.block8 import Block8, Rows8

    if "ctx" not in _kept:
        _kept["ctx"] = capi.Context(torch.cuda.current_device())
    ctx = s["ctx"] = _kept["ctx"]
    kind = s["kind"]
    if "rows" in s:
        ptr = np.zeros(_blocks(s["rows"]) + 1, dtype=np.int64)
        np.cumsum(np.bincount(s["block_row"].cpu().numpy(), minlength=len(ptr) - 1), out=ptr[1:])
        s["matrix"] = Block8(ctx, s["rows"], s["cols"], ptr, s["block_col"].cpu().numpy().astype(np.uint32), transposed=kind in ("backward", "step"))
        torch.cuda.synchronize()  # (the library's calls run on its context's stream)
        if "values" in s:
            s["matrix"].set_values(s["values"].data_ptr(), "f32")
    if kind == "update":
        s["out"] = torch.empty_like(s["master"])
    if "tokens" in case:
        t, dtype = case["tokens"], TYPES[case["dtype"]]
        if kind != "single":
            s["saved"] = Rows8(ctx, t, s["x"].shape[1])
        if kind == "checkpoint":
            s["out"] = torch.empty(t, case["cols"], dtype=dtype, device="cuda")
        if kind in ("single", "product", "step"):
            s["y"] = torch.empty(t, case["rows"], dtype=dtype, device="cuda")
        if kind in ("backward", "step"):
            s["grads"] = Rows8(ctx, t, case["rows"])
            s["dx"] = torch.empty(t, case["cols"], dtype=dtype, device="cuda")
            s["da"] = torch.empty(s["master"].shape, dtype=torch.float32, device="cuda")
        if kind == "backward":
            s["saved"].quantize(s["x"].data_ptr(), t, s["dtype"], s["x"].stride(0))
    ctx.synchronize()


_kept = {}  # the one context that a program has per GPU


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    kind, dtype = s["kind"], s.get("dtype")
    if kind == "update":
        s["matrix"].set_values(s["master"].data_ptr(), "f32")
        s["matrix"].get_values(s["out"].data_ptr())
        return {"values": s["out"]}
    x = s["x"]
    tokens = x.shape[0]
    if kind == "single":
        s["matrix"].apply(x.data_ptr(), tokens, dtype, s["y"].data_ptr(), dtype)
        return {"y": s["y"]}
    if kind == "checkpoint":
        s["saved"].quantize(x.data_ptr(), tokens, dtype, x.stride(0))
        s["saved"].restore(s["out"].data_ptr(), dtype)
        return {"x": s["out"]}
    if kind == "product":
        s["saved"].quantize(x.data_ptr(), tokens, dtype)
        s["matrix"].product(s["saved"], s["y"].data_ptr(), dtype)
        return {"y": s["y"]}
    dy = s["dy"]
    if kind == "step":
        s["matrix"].set_values(s["master"].data_ptr(), "f32")
        s["saved"].quantize(x.data_ptr(), tokens, dtype)
        s["matrix"].product(s["saved"], s["y"].data_ptr(), dtype)
    s["matrix"].gradient(s["saved"], dy.data_ptr(), dtype, s["da"].data_ptr())
    s["grads"].quantize(dy.data_ptr(), tokens, dtype)
    s["matrix"].product(s["grads"], s["dx"].data_ptr(), dtype, transposed=True)
    return {"y": s["y"], "dx": s["dx"], "da": s["da"]} if kind == "step" else {"dx": s["dx"], "da": s["da"]}


def _eight_bits(x, width):
    """What e4m3 with a scale for each `width` columns stands for, in 32 bits. An element that is not finite becomes NaN and has no
    say in the scale."""
    rows, cols = x.shape
    f = torch.nn.functional.pad(x.float(), (0, -cols % width)).reshape(rows, -1, width)
    most = torch.where(f.isfinite(), f.abs(), 0.0).amax(-1, keepdim=True)
    fraction, exponent = torch.frexp(most)  # 448 = 0.875 * 2^9
    k = torch.clamp(exponent - 9 + (fraction > 0.875), min=-126)
    q = (f * _power(-k)).to(torch.float8_e4m3fn)
    return (q.float() * _power(k)).reshape(rows, -1)[:, :cols]


def _power(k):
    """2^k, exactly (pow is not), for -126 <= k <= 126."""
    return ((k + 127) << 23).to(torch.int32).view(torch.float32)


def _dense(s, values):
    """The matrix, zero where no block is stored, to whole blocks."""
    a = torch.zeros(_blocks(s["rows"]), _blocks(s["cols"]), BLOCK, BLOCK, device="cuda", dtype=values.dtype)
    a[s["block_row"], s["block_col"]] = values
    return a.transpose(1, 2).reshape(_blocks(s["rows"]) * BLOCK, -1)[: s["rows"], : s["cols"]]


def _stored(s, full):
    """The stored blocks of an n_rows x n_cols matrix."""
    full = torch.nn.functional.pad(full, (0, -s["cols"] % BLOCK, 0, -s["rows"] % BLOCK))
    return full.reshape(_blocks(s["rows"]), BLOCK, -1, BLOCK).transpose(1, 2)[s["block_row"], s["block_col"]]


def _plain(s):
    kind, dtype = s["kind"], TYPES.get(s.get("dtype"))
    if kind == "checkpoint":
        return {"x": _eight_bits(s["x"], BLOCK).to(dtype)}
    if kind in ("update", "step"):
        n = s["master"].shape[0]
        values = _eight_bits(s["master"].reshape(n, -1), BLOCK * BLOCK).reshape(n, BLOCK, BLOCK)
        if kind == "update":
            return {"values": values}
    else:
        values = s["values"]
    a = _dense(s, values)
    x = _eight_bits(s["x"], BLOCK)
    if kind in ("single", "product"):
        return {"y": (x @ a.T).to(dtype)}
    grads = {"dx": (_eight_bits(s["dy"], BLOCK) @ a).to(dtype), "da": _stored(s, s["dy"].float().T @ x)}
    return {"y": (x @ a.T).to(dtype), **grads} if kind == "step" else grads


# ---- from the definition, in 64 bits -----------------------------------------------------------------------------------
def _rounded(v):
    """To the nearest e4m3 (ties to the even one), |v| <= 448: four significant bits, and a step of 2^-9 below 2^-6."""
    step = torch.exp2((torch.frexp(v).exponent - 1).clamp(min=-6).double() - 3.0)
    return torch.round(v / step) * step


def _stands_for(groups):
    """groups: [n, width] in 64 bits, a scale each."""
    most = groups.abs().amax(1, keepdim=True)
    fraction, exponent = torch.frexp(most / 448.0)
    scale = torch.exp2((exponent - (fraction == 0.5).int()).clamp(min=-126).double())
    return _rounded(groups / scale) * scale


def _rows_stand_for(x):
    full = torch.zeros(x.shape[0], _blocks(x.shape[1]) * BLOCK, dtype=torch.float64, device=x.device)
    full[:, : x.shape[1]] = x
    return _stands_for(full.reshape(-1, BLOCK)).reshape(full.shape)


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "checkpoint":
        return {"x": _rows_stand_for(s["x"])[:, : case["cols"]]}
    n = s["master"].shape[0]
    blocks = _stands_for(s["master"].double().reshape(n, -1)).reshape(n, BLOCK, BLOCK)
    if kind == "update":
        return {"values": blocks}
    whole = torch.zeros(_blocks(s["rows"]) * BLOCK, _blocks(s["cols"]) * BLOCK, dtype=torch.float64, device="cuda")
    tiles = whole.unflatten(0, (-1, BLOCK)).unflatten(2, (-1, BLOCK))  # block row, row, block column, column
    tiles.permute(0, 2, 1, 3)[s["block_row"], s["block_col"]] = blocks
    x = _rows_stand_for(s["x"])
    out = {}
    if kind != "backward":
        out["y"] = torch.einsum("tc,rc->tr", x, whole)[:, : s["rows"]]
    if kind in ("backward", "step"):
        out["dx"] = torch.einsum("tr,rc->tc", _rows_stand_for(s["dy"]), whole)[:, : s["cols"]]
        dy = torch.zeros(case["tokens"], whole.shape[0], dtype=torch.float64, device="cuda")
        dy[:, : s["rows"]] = s["dy"]
        da = torch.einsum("tr,tc->rc", dy, x).unflatten(0, (-1, BLOCK)).unflatten(2, (-1, BLOCK)).permute(0, 2, 1, 3)
        out["da"] = da[s["block_row"], s["block_col"]]
    return out


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------
def work(case):
    """Each input read once and each output written once, in the types the case has them in; the stored blocks by their expected
    number, a byte an element where 8 bits are what is kept; two operations for each product that a stored element takes part in. What
    is kept in 8 bits and needed again is written and read once."""
    kind = case["kind"]
    size = {"f32": 4, "f16": 2, "bf16": 2}.get(case.get("dtype"), 4)
    tokens, rows, cols = case.get("tokens", 0), case.get("rows", 0), case.get("cols", 0)
    if kind == "checkpoint":
        return {"bytes": 2.0 * tokens * cols * (size + 1), "flops": 0.0}
    stored = rows * cols * case["density"]
    if kind == "update":
        return {"bytes": stored * (4 + 1 + 1 + 4), "flops": 0.0}
    forward = {"bytes": stored + size * tokens * (rows + cols), "flops": 2.0 * tokens * stored}
    if kind in ("single", "product"):
        return forward
    backward = {"bytes": stored + 4 * stored + size * tokens * (rows + cols) + tokens * cols, "flops": 4.0 * tokens * stored}
    if kind == "backward":
        return backward
    return {"bytes": 4 * stored + forward["bytes"] + backward["bytes"] + tokens * cols, "flops": forward["flops"] + backward["flops"]}
