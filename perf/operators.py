"""Measured cases of the expert-routing operators: ``topk_route``, ``route_csr``, ``segment_matmul``, ``quantize_fp8`` and
``segment_matmul_fp8``, each with its plain form in elementary torch operations and its definition in 64 bits.

Together they are one layer of routed experts (or of typed relations): every row is given to its best experts, the
(row, expert) pairs become a CSR structure with one segment per expert, each segment is multiplied by its own matrix,
and for serving the products run on 8-bit values with one scale for each block of 128.
"""
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 128          # values that share one scale along the reduced dimension
FP8_MAX = 448.0      # largest finite value of float8_e4m3fn


# ---- cases -------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # One step of a small serving batch: latency of the router alone.
        dict(name="route_decode", op="route", tokens=8, experts=64, k=2, score="softmax", bias=False, groups=1, kept=1,
             renormalize=True, dtype="bf16", backward=False),
        # A training micro-batch with balancing bias and expert groups; the router's logits are kept in fp32.
        dict(name="route_groups", op="route", tokens=4099, experts=256, k=8, score="sigmoid", bias=True, groups=8, kept=4,
             renormalize=True, dtype="fp32", backward=True),
        # A large training batch, or the nodes of a large graph given to experts.
        dict(name="route_batch", op="route", tokens=131072, experts=128, k=8, score="softmax", bias=False, groups=1, kept=1,
             renormalize=True, dtype="bf16", backward=True),
        # The dispatch structure of one serving step.
        dict(name="plan_decode", op="plan", tokens=64, experts=128, k=8, dropped=0.0),
        # The dispatch structure of a large batch, some pairs dropped over capacity (expert -1).
        dict(name="plan_batch", op="plan", tokens=131072, experts=256, k=8, dropped=0.03),
        # Experts' products of one serving step: a row or two for each expert, every weight is read.
        dict(name="products_decode", op="products", rows=96, behind=0, segments=64, width=2048, out=1024, layout="nk",
             dtype="bf16", backward=False),
        # Experts' products of a training step, forward and both gradients, ragged segments, rows behind the last one.
        dict(name="products_train", op="products", rows=32768, behind=37, segments=32, width=2048, out=1024, layout="kn",
             dtype="bf16", backward=True),
        # Typed linear layer of a relational graph in fp32 (feature width of the repository's benchmark).
        dict(name="products_relations", op="products", rows=200003, behind=0, segments=13, width=256, out=256, layout="kn",
             dtype="fp32", backward=True),
        # Activations of a prompt on their way into an 8-bit product: one scale per row and 128 columns.
        dict(name="quantize_rows", op="quantize", count=1, rows=16381, width=4096, block_rows=1, dtype="bf16"),
        # Weights of a layer's experts on loading: one scale per tile of 128 x 128.
        dict(name="quantize_experts", op="quantize", count=64, rows=1024, width=2048, block_rows=128, dtype="bf16"),
        # 8-bit experts' products of one serving step.
        dict(name="fp8_decode", op="fp8", rows=64, segments=32, width=2048, out=2048, scales="power", dtype="bf16"),
        # 8-bit experts' products of a batch of prompts.
        dict(name="fp8_prompt", op="fp8", rows=65536, segments=16, width=4096, out=2048, scales="any", dtype="bf16"),
    ]


def _log(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(["route", "plan", "products", "products", "quantize", "fp8"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * rng.randint(2, 256 // groups)
        kept = rng.randint(1, groups)
        return dict(op=op, tokens=_log(rng, 1, 65536), experts=experts, k=rng.randint(1, min(16, kept * (experts // groups))),
                    score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups, kept=kept,
                    renormalize=rng.random() < 0.7, dtype=rng.choice(["bf16", "fp16", "fp32"]), backward=rng.random() < 0.7)
    if op == "plan":
        return dict(op=op, tokens=_log(rng, 1, 131072), experts=rng.randint(1, 512), k=rng.randint(1, 8),
                    dropped=rng.choice([0.0, 0.0, 0.05]))
    if op == "products":
        kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        # any width in one draw of four; whole 16-byte vectors otherwise, as feature widths mostly are
        step = 1 if rng.random() < 0.25 else 8
        top = 512 if kind == "fp32" or step == 1 else 2048
        width, out = (max(1, _log(rng, 16, top) // step) * step for _ in range(2))
        return dict(op=op, rows=_log(rng, 1, 32768), behind=rng.choice([0, 0, rng.randint(1, 300)]), segments=rng.randint(1, 64),
                    width=width, out=out, layout=rng.choice(["kn", "nk"]), dtype=kind, backward=rng.random() < 0.6)
    if op == "quantize":
        block_rows = rng.choice([1, 128])
        return dict(op=op, count=rng.choice([1, 1, rng.randint(2, 8)]), rows=_log(rng, 1, 4096), width=_log(rng, 16, 4096),
                    block_rows=block_rows, dtype=rng.choice(["bf16", "fp16", "fp32"]))
    return dict(op=op, rows=_log(rng, 1, 16384), segments=rng.choice([0, rng.randint(1, 32)]), width=16 * _log(rng, 4, 256),
                out=8 * _log(rng, 4, 256), scales=rng.choice(["power", "any"]), dtype=rng.choice(["bf16", "fp16", "fp32"]))


def _lengths(rows, segments, seed):
    """Segment lengths that add up to `rows`: uneven as routing is, one segment in eight empty where there are several."""
    r = np.random.RandomState(seed % (1 << 31))
    share = r.dirichlet(np.full(segments, 8.0))
    if segments >= 8:
        share[r.permutation(segments)[:segments // 8]] = 0.0
        share /= share.sum()
    return r.multinomial(rows, share)


def _pointers(lengths):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)).cuda()


# ---- inputs ------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    s = dict(case)
    op = case["op"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if op == "route":
        t = DTYPES[case["dtype"]]
        s["logits"] = (normal(case["tokens"], case["experts"]) * 1.5).to(t).requires_grad_(case["backward"])
        s["shift"] = normal(case["experts"]) * 0.05 if case["bias"] else None
        s["grad"] = normal(case["tokens"], case["k"]).to(t)
    elif op == "plan":
        # k different experts a row, some more popular than others
        keys = torch.rand(case["tokens"], case["experts"], generator=g, device="cuda") + \
            0.5 * torch.rand(case["experts"], generator=g, device="cuda")
        k = min(case["k"], case["experts"])
        index = keys.topk(k, dim=1).indices
        drop = torch.rand(index.shape, generator=g, device="cuda") < case["dropped"]
        s["index"] = torch.where(drop, torch.full_like(index, -1), index)
    elif op == "products":
        t = DTYPES[case["dtype"]]
        lengths = _lengths(case["rows"], case["segments"], seed)
        s["indptr"], s["longest"] = _pointers(lengths), int(lengths.max())
        s["src"] = normal(case["rows"] + case["behind"], case["width"]).to(t).requires_grad_(case["backward"])
        e, k, n = case["segments"], case["width"], case["out"]
        weight = (normal(e, n, k) if case["layout"] == "nk" else normal(e, k, n)) * k ** -0.5
        s["weight"] = weight.to(t).requires_grad_(case["backward"])
        s["grad"] = normal(case["rows"] + case["behind"], n).to(t) if case["backward"] else None
    elif op == "quantize":
        t = DTYPES[case["dtype"]]
        x = normal(case["count"], case["rows"], case["width"]) * normal(case["count"], case["rows"], 1).exp()
        s["src"] = (x if case["count"] > 1 else x[0]).to(t)
    else:
        groups = max(1, case["segments"])
        lengths = _lengths(case["rows"], groups, seed)
        s["indptr"] = _pointers(lengths) if case["segments"] else None
        s["longest"] = int(lengths.max())
        s["src"], s["src_scale"] = _eight_bits(normal(case["rows"], case["width"]), 1, case["scales"])
        weight = normal(groups, case["out"], case["width"]) * case["width"] ** -0.5
        s["weight"], s["weight_scale"] = _eight_bits(weight if case["segments"] else weight[0], BLOCK, case["scales"])
    return s


def _eight_bits(x, block_rows, scales):
    """8-bit values of x and their scales, as a checkpoint or an earlier layer hands them over."""
    top = _blocks(x.abs(), block_rows).amax((-3, -1))
    scale = _power(top) if scales == "power" else torch.where(top > 0, top / FP8_MAX, torch.ones_like(top))
    return (x / _spread(scale, block_rows, x.shape)).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn), scale


# ---- plain forms -------------------------------------------------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    return {"route": _route, "plan": _plan, "products": _products, "quantize": _quantize, "fp8": _fp8}[s["op"]](s)


def _route(s):
    """Scores of all experts; the best groups by the sum of their two best biased scores; the best k experts of these."""
    tokens, experts, k, groups = s["tokens"], s["experts"], s["k"], s["groups"]
    logits = s["logits"].detach()
    # the choice in 64 bits: scores that differ by less than fp32 tells apart decide it
    fine = logits.double()
    chosen_by = torch.softmax(fine, 1) if s["score"] == "softmax" else torch.sigmoid(fine)
    if s["bias"]:
        chosen_by = chosen_by + s["shift"].double()
    if groups > 1:
        best = chosen_by.view(tokens, groups, -1).sort(dim=2, descending=True).values[:, :, :2].sum(2)
        order = best.sort(dim=1, descending=True, stable=True).indices[:, :s["kept"]]
        open_groups = torch.zeros(tokens, groups, dtype=torch.bool, device=logits.device).scatter_(1, order, True)
        chosen_by = chosen_by.masked_fill(~open_groups.repeat_interleave(experts // groups, 1), -float("inf"))
    index = chosen_by.sort(dim=1, descending=True, stable=True).indices[:, :k].contiguous()
    score = torch.softmax(logits.float(), 1) if s["score"] == "softmax" else torch.sigmoid(logits.float())
    picked = score.gather(1, index)
    total = picked.sum(1, keepdim=True)
    weight = picked / total if s["renormalize"] else picked
    if not s["backward"]:
        return {"weight": weight.to(logits.dtype), "index": index}
    grad = s["grad"].float()
    if s["renormalize"]:
        grad = (grad - (grad * weight).sum(1, keepdim=True)) / total
    back = torch.zeros_like(score).scatter_(1, index, grad)
    if s["score"] == "softmax":
        back = score * (back - (back * score).sum(1, keepdim=True))
    else:
        back = back * score * (1 - score)
    return {"weight": weight.to(logits.dtype), "index": index, "grad_logits": back.to(logits.dtype)}


def _plan(s):
    """Pairs in the order of their experts, pairs of one expert in the order they came, dropped pairs last."""
    label = s["index"].reshape(-1)
    label = torch.where((label >= 0) & (label < s["experts"]), label, torch.full_like(label, s["experts"]))
    perm = torch.sort(label, stable=True).indices
    counts = torch.bincount(label, minlength=s["experts"] + 1)[:s["experts"]]
    indptr = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    position = torch.empty_like(perm).scatter_(0, perm, torch.arange(perm.numel(), device=perm.device))
    return {"indptr": indptr, "perm": perm, "position": position.view(s["index"].shape)}


def _slots(s, rows):
    """Where each row stands among [segment, place within the segment], rows behind the last segment marked."""
    row = torch.arange(rows, device=s["indptr"].device)
    segment = torch.searchsorted(s["indptr"], row, right=True) - 1
    inside = segment < s["indptr"].numel() - 1
    segment = segment.clamp(max=s["indptr"].numel() - 2)
    return segment, (row - s["indptr"][segment]).clamp(max=max(0, s["longest"] - 1)), inside


def _padded(x, slots, segments, longest):
    segment, place, inside = slots
    out = x.new_zeros(segments, longest, x.size(1))
    out[segment[inside], place[inside]] = x[inside]
    return out


def _unpadded(x, slots):
    segment, place, inside = slots
    return x[segment, place] * inside.unsqueeze(1)


def _products(s):
    """out[r] = src[r] @ weight[e] for the rows r of segment e; both gradients; 0 in rows of no segment."""
    src, weight = s["src"].detach(), s["weight"].detach().float()
    if s["layout"] == "nk":
        weight = weight.transpose(1, 2)
    slots = _slots(s, src.size(0))
    x = _padded(src.float(), slots, s["segments"], s["longest"])
    out = _unpadded(torch.bmm(x, weight), slots).to(src.dtype)
    if not s["backward"]:
        return {"out": out}
    grad = _padded(s["grad"].float(), slots, s["segments"], s["longest"])
    grad_src = _unpadded(torch.bmm(grad, weight.transpose(1, 2)), slots).to(src.dtype)
    if s["layout"] == "nk":
        grad_weight = torch.bmm(grad.transpose(1, 2), x)
    else:
        grad_weight = torch.bmm(x.transpose(1, 2), grad)
    return {"out": out, "grad_src": grad_src, "grad_weight": grad_weight.to(src.dtype)}


def _blocks(x, block_rows):
    """x as [..., row blocks, rows of a block, column blocks, columns of a block], zeros past the edges."""
    rows, width = x.shape[-2:]
    down, across = -(-rows // block_rows), -(-width // BLOCK)
    x = torch.nn.functional.pad(x, (0, across * BLOCK - width, 0, down * block_rows - rows))
    return x.reshape(*x.shape[:-2], down, block_rows, across, BLOCK)


def _spread(scale, block_rows, shape):
    return scale.repeat_interleave(block_rows, -2)[..., :shape[-2], :].repeat_interleave(BLOCK, -1)[..., :shape[-1]]


def _power(top):
    """The smallest power of two that brings `top` to at most 448 = 0.875 * 2^9; 1 for a block of zeros."""
    part, exponent = torch.frexp(top)
    exponent = (exponent - 9 + (part > 0.875)).clamp(min=-126)
    return torch.where(top > 0, torch.ldexp(torch.ones_like(top), exponent), torch.ones_like(top))


def _quantize(s):
    x = s["src"].float()
    scale = _power(_blocks(x.abs(), s["block_rows"]).amax((-3, -1)))
    values = (x / _spread(scale, s["block_rows"], x.shape)).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return {"values": values, "scale": scale}


def _fp8(s):
    src = s["src"].float() * _spread(s["src_scale"], 1, s["src"].shape)
    weight = s["weight"].float() * _spread(s["weight_scale"], BLOCK, s["weight"].shape)
    if not s["segments"]:
        return {"out": torch.mm(src, weight.t()).to(DTYPES[s["dtype"]])}
    slots = _slots(s, src.size(0))
    x = _padded(src, slots, s["segments"], s["longest"])
    return {"out": _unpadded(torch.bmm(x, weight.transpose(1, 2)), slots).to(DTYPES[s["dtype"]])}


# ---- the framework's calls ---------------------------------------------------------------------------------------------

def _package():
    here = os.path.join(os.getcwd(), "ops-gnn_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import ops_gnn

    return ops_gnn


def _run_own(s):
    ops_gnn = _package()
    op = s["op"]
    if op == "route":
        weight, index = ops_gnn.topk_route(s["logits"], s["k"], score=s["score"], bias=s["shift"], groups=s["groups"],
                                           kept_groups=s["kept"], renormalize=s["renormalize"])
        if not s["backward"]:
            return {"weight": weight, "index": index}
        return {"weight": weight, "index": index, "grad_logits": torch.autograd.grad(weight, s["logits"], s["grad"])[0]}
    if op == "plan":
        indptr, perm, position = ops_gnn.route_csr(s["index"], s["experts"])
        return {"indptr": indptr, "perm": perm, "position": position}
    if op == "products":
        weight = s["weight"].transpose(1, 2) if s["layout"] == "nk" else s["weight"]
        out = ops_gnn.segment_matmul(s["src"], s["indptr"], weight)
        if not s["backward"]:
            return {"out": out}
        grad_src, grad_weight = torch.autograd.grad(out, (s["src"], s["weight"]), s["grad"])
        return {"out": out, "grad_src": grad_src, "grad_weight": grad_weight}
    if op == "quantize":
        values, scale = ops_gnn.quantize_fp8(s["src"], block_rows=s["block_rows"])
        return {"values": values, "scale": scale}
    out = ops_gnn.segment_matmul_fp8(s["src"], s["src_scale"], s["weight"], s["weight_scale"], indptr=s["indptr"],
                                     out_dtype=DTYPES[s["dtype"]])
    return {"out": out}


# ---- what a pass cannot do without -------------------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "route":
        size, t, e, k = DTYPES[case["dtype"]].itemsize, case["tokens"], case["experts"], case["k"]
        back = case["backward"]
        return {"bytes": t * e * size + t * k * (size + 8) + (4 * e if case["bias"] else 0) + (t * (k + e) * size if back else 0),
                "flops": t * e * (8 if back else 4)}
    if op == "plan":
        pairs = case["tokens"] * min(case["k"], case["experts"])
        return {"bytes": pairs * 24 + 8 * (case["experts"] + 1), "flops": 0}
    if op == "products":
        size, e, k, n = DTYPES[case["dtype"]].itemsize, case["segments"], case["width"], case["out"]
        rows = case["rows"] + case["behind"]
        forward = rows * (k + n) + e * k * n
        return {"bytes": size * (forward + (rows * (n + k) + e * k * n if case["backward"] else 0)) + 8 * (e + 1),
                "flops": 2 * case["rows"] * k * n * (3 if case["backward"] else 1)}
    if op == "quantize":
        n, size = case["count"] * case["rows"] * case["width"], DTYPES[case["dtype"]].itemsize
        scales = case["count"] * -(-case["rows"] // case["block_rows"]) * -(-case["width"] // BLOCK)
        return {"bytes": n * (size + 1) + 4 * scales, "flops": 2 * n}
    e, k, n, rows = max(1, case["segments"]), case["width"], case["out"], case["rows"]
    scales = -(-k // BLOCK) * (rows + e * -(-n // BLOCK))
    return {"bytes": rows * k + e * n * k + 4 * scales + rows * n * DTYPES[case["dtype"]].itemsize, "flops": 2 * rows * k * n}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "plan":
        return None
    if op == "route":
        return _exact_route(s)
    if op == "quantize":
        return _exact_quantize(s)
    if op == "fp8":
        src, weight = _stands_for(s["src"], s["src_scale"], 1), _stands_for(s["weight"], s["weight_scale"], BLOCK)
        if not case["segments"]:
            return {"out": src @ weight.mT}
        return {"out": _each(src, s["indptr"], weight.mT)}
    src, weight = s["src"].detach().double(), s["weight"].detach().double()
    weight = weight.mT if case["layout"] == "nk" else weight
    out = _each(src, s["indptr"], weight)
    if not case["backward"]:
        return {"out": out}
    grad = s["grad"].double()
    ends = s["indptr"].tolist()
    grad_weight = torch.stack([src[a:b].mT @ grad[a:b] for a, b in zip(ends, ends[1:])])
    return {"out": out, "grad_src": _each(grad, s["indptr"], weight.mT),
            "grad_weight": grad_weight.mT if case["layout"] == "nk" else grad_weight}


def _each(x, indptr, matrices):
    out = x.new_zeros(x.size(0), matrices.size(2))
    ends = indptr.tolist()
    for e, (a, b) in enumerate(zip(ends, ends[1:])):
        out[a:b] = x[a:b] @ matrices[e]
    return out


def _stands_for(values, scale, block_rows):
    value = values.double()
    row = torch.arange(value.size(-2), device=value.device) // block_rows
    column = torch.arange(value.size(-1), device=value.device) // BLOCK
    return value * scale.double()[..., row, :][..., column]


def _exact_route(s):
    x = s["logits"].detach().double()
    t, e, k = s["tokens"], s["experts"], s["k"]
    z = (x - x.amax(1, keepdim=True)).exp()
    score = z / z.sum(1, keepdim=True) if s["score"] == "softmax" else 1 / (1 + (-x).exp())
    by = score if s["shift"] is None else score + s["shift"].double()
    size = e // s["groups"]
    if s["groups"] > 1:
        # a group's rank: how many groups are better, or as good and before it
        in_group = by.view(t, s["groups"], size)
        first = in_group.max(2)
        rest = in_group.scatter(2, first.indices.unsqueeze(2), -float("inf")).amax(2)
        best = first.values + rest
        number = torch.arange(s["groups"], device=x.device)
        ahead = (best.unsqueeze(1) > best.unsqueeze(2)) | \
            ((best.unsqueeze(1) == best.unsqueeze(2)) & (number.view(1, 1, -1) < number.view(1, -1, 1)))
        keep = ahead.sum(2) < s["kept"]
        by = torch.where(keep.unsqueeze(2).expand(t, s["groups"], size).reshape(t, e), by, by.new_tensor(-float("inf")))
    index = torch.empty(t, k, dtype=torch.int64, device=x.device)
    for j in range(k):
        top = by.amax(1, keepdim=True)
        first = torch.where(by == top, torch.arange(e, device=x.device), e).amin(1)
        index[:, j] = first
        by = by.scatter(1, first.unsqueeze(1), -float("inf"))
    mine = torch.gather(score, 1, index)
    total = mine.sum(1, keepdim=True) if s["renormalize"] else torch.ones_like(mine[:, :1])
    weight = mine / total
    if not s["backward"]:
        return {"weight": weight, "index": None}
    g = s["grad"].double()
    if s["renormalize"]:
        g = g / total - (g * mine).sum(1, keepdim=True) / total ** 2
    if s["score"] == "softmax":
        back = -score * (g * mine).sum(1, keepdim=True)
        back = back.scatter_add(1, index, g * mine)
    else:
        back = torch.zeros_like(score).scatter_add(1, index, g * mine * (1 - mine))
    return {"weight": weight, "index": None, "grad_logits": back}


def _exact_quantize(s):
    x = s["src"].double()
    x3 = x if x.dim() == 3 else x.unsqueeze(0)
    c, r, w = x3.shape
    row = torch.arange(r, device=x.device) // s["block_rows"]
    column = torch.arange(w, device=x.device) // BLOCK
    down, across = int(row[-1]) + 1, int(column[-1]) + 1
    block = (row.view(-1, 1) * across + column.view(1, -1)).reshape(-1)
    top = x.new_zeros(c, down * across).scatter_reduce_(1, block.expand(c, -1), x3.abs().reshape(c, -1), "amax")
    exponent = torch.ceil(torch.log2(top / FP8_MAX) - 1e-13).clamp(min=-126)
    scale = torch.where(top > 0, torch.exp2(exponent), torch.ones_like(top))
    y = x3 / scale[:, block].view(c, r, w)
    # nearest multiple of the step at |y|: 2^(exponent - 3), no finer than 2^-9; ties to even
    step = torch.exp2((torch.frexp(y.abs()).exponent - 1).clamp(min=-6).double() - 3)
    y = torch.round(y / step) * step
    scale = scale.view(c, down, across)
    return {"values": y if x.dim() == 3 else y[0], "scale": scale if x.dim() == 3 else scale[0]}
