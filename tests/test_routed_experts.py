"""Routed experts: topk_route, route_csr, segment_matmul, quantize_fp8, segment_matmul_fp8 and a layer made of them, against
plain float64 restatements on the CPU.

Bounds.  A result of 16 or 32 bits is rounded once, by at most eps / 2 of its value.  A sum of n products held in fp32 is off
by at most n * 2^-23 of the sum of their magnitudes, whatever its order and whether an addition rounds or cuts off (2^-23 is a
whole step of fp32).  Scores: exp and the division are good to a few steps of fp32, their sum over E experts to E half steps.
"""
import ctypes
import math

import pytest
import torch

from conftest import requires_gpu

STEP = 2.0 ** -23


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- plain restatements --------------------------------------------------------------------------------------------------

def _plain_scores(logits, score):
    x = logits.double()
    if score == "sigmoid":
        return torch.sigmoid(x)
    top = x.max(1, keepdim=True).values
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    z = torch.exp(x - top)
    total = z.sum(1, keepdim=True)
    return torch.where(total == 0, torch.zeros_like(z), z / total)


def _plain_choice(logits, k, score, bias, groups, kept, group_top):
    """Row by row, as the definition says it; returns a list of k experts per row."""
    s = _plain_scores(logits, score)
    experts = logits.size(1)
    size = experts // groups
    chosen = []
    for r in range(logits.size(0)):
        row = [float(v) for v in s[r]]
        if bias is None and (groups == 1 or group_top == 1):
            row = [float(v) if not math.isnan(row[j]) else math.nan for j, v in enumerate(logits[r].double())]
        if bias is not None:
            row = [v + float(b) for v, b in zip(row, bias.double())]
        row = [-math.inf if float(l) == -math.inf or math.isnan(v) else v for v, l in zip(row, logits[r])]
        rank = sorted(range(groups), key=lambda g: (-sum(sorted(row[g * size:(g + 1) * size], reverse=True)[:group_top]), g))
        open_groups = set(rank[:kept])
        order = sorted((j for j in range(experts) if j // size in open_groups), key=lambda j: (-row[j], j))
        chosen.append(order[:k])
    return torch.tensor(chosen, dtype=torch.int64).reshape(logits.size(0), k)


def _plain_weight(logits, index, score, renormalize, scale):
    if score == "softmax" and renormalize:
        # the sum over all experts cancels; leaving it out keeps float64 rounding off the experts not chosen
        return _plain_scores(logits.gather(1, index), score) * scale
    s = _plain_scores(logits, score).gather(1, index)
    if renormalize:
        total = s.sum(1, keepdim=True)
        s = torch.where(total == 0, torch.zeros_like(s), s / total)
    return s * scale


def _plain_matmul(src, ptr, weight):
    out = torch.zeros(src.size(0), weight.size(2), dtype=torch.float64)
    for e in range(weight.size(0)):
        out[ptr[e]:ptr[e + 1]] = src[ptr[e]:ptr[e + 1]].double() @ weight[e].double()
    return out


def _plain_weight_grad(src, ptr, grad):
    return torch.stack([src[ptr[e]:ptr[e + 1]].double().t() @ grad[ptr[e]:ptr[e + 1]].double() for e in range(len(ptr) - 1)]) \
        if len(ptr) > 1 else torch.zeros(0, src.size(1), grad.size(1), dtype=torch.float64)


def _within(actual, expected, magnitude, terms, what):
    """|actual - expected| <= eps / 2 * |expected| + terms * 2^-23 * magnitude, plus half the smallest subnormal step."""
    assert actual.shape == expected.shape, what
    info = torch.finfo(actual.dtype)
    got, want = actual.detach().cpu().double(), expected.double()
    assert torch.isfinite(got).all(), what + ": unexpected NaN or infinity"
    slack = info.eps / 2 * want.abs() + terms * STEP * magnitude.double() * (1 + info.eps) + info.smallest_normal * info.eps
    over = ((got - want).abs() / slack.clamp(min=1e-300)).max().item() if got.numel() else 0.0
    assert over <= 1.0, f"{what}: {over:.2f} times the bound"


def _pointers(lengths, first=0):
    return torch.tensor([first] + list(first + torch.tensor(lengths, dtype=torch.int64).cumsum(0))) if len(lengths) \
        else torch.tensor([first])


# ---- refusals (no GPU) ---------------------------------------------------------------------------------------------------

def test_topk_route_refuses():
    from ops_gnn import topk_route

    x = torch.zeros(4, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        topk_route(x, 2)
    with pytest.raises(TypeError, match="torch.Tensor"):
        topk_route([1.0], 1)
    with pytest.raises(TypeError, match="float16"):
        topk_route(x.double(), 2)
    with pytest.raises(ValueError, match="dimension"):
        topk_route(torch.tensor(1.0), 1)
    with pytest.raises(ValueError, match="softmax"):
        topk_route(x, 2, score="tanh")
    for bad in (0, 17):
        with pytest.raises(ValueError, match="k must be"):
            topk_route(x, bad)
    with pytest.raises(TypeError, match="k must be an int"):
        topk_route(x, True)
    with pytest.raises(ValueError, match="divide"):
        topk_route(x, 2, groups=3)
    with pytest.raises(ValueError, match="kept_groups"):
        topk_route(x, 2, groups=4, kept_groups=5)
    with pytest.raises(ValueError, match="k must be"):
        topk_route(x, 5, groups=4, kept_groups=1)
    with pytest.raises(ValueError, match="group_top"):
        topk_route(x, 2, groups=16, group_top=2)
    with pytest.raises(ValueError, match="group_top"):
        topk_route(x, 2, groups=4, group_top=3)
    with pytest.raises(ValueError, match="experts"):
        topk_route(torch.zeros(1, 1025), 1)
    with pytest.raises(ValueError, match="k must be"):
        topk_route(torch.zeros(1, 64), 33)
    with pytest.raises(TypeError, match="bias"):
        topk_route(x, 2, bias=torch.zeros(16, dtype=torch.float64))
    with pytest.raises(ValueError, match="bias"):
        topk_route(x, 2, bias=torch.zeros(15))


def test_route_csr_refuses():
    from ops_gnn import route_csr

    x = torch.zeros(4, 2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        route_csr(x, 4)
    with pytest.raises(TypeError, match="int32"):
        route_csr(x.float(), 4)
    with pytest.raises(TypeError, match="torch.Tensor"):
        route_csr([1], 4)
    with pytest.raises(TypeError, match="num_experts"):
        route_csr(x, 4.0)
    for bad in (0, 4097):
        with pytest.raises(ValueError, match="num_experts"):
            route_csr(x, bad)


def test_segment_matmul_refuses():
    from ops_gnn import segment_matmul

    src, ptr, weight = torch.zeros(4, 8), torch.tensor([0, 4]), torch.zeros(1, 8, 3)
    with pytest.raises(RuntimeError, match="CUDA"):
        segment_matmul(src, ptr, weight)
    with pytest.raises(TypeError, match="src"):
        segment_matmul([1], ptr, weight)
    with pytest.raises(TypeError, match="weight"):
        segment_matmul(src, ptr, None)
    with pytest.raises(TypeError, match="dtype"):
        segment_matmul(src.double(), ptr, weight.double())
    with pytest.raises(TypeError, match="match"):
        segment_matmul(src, ptr, weight.half())
    with pytest.raises(TypeError, match="indptr"):
        segment_matmul(src, ptr.float(), weight)
    with pytest.raises(ValueError, match="2-D"):
        segment_matmul(src[0], ptr, weight)
    with pytest.raises(ValueError, match="3-D"):
        segment_matmul(src, ptr, weight[0])
    with pytest.raises(ValueError, match="size"):
        segment_matmul(src, ptr, weight[:, :7])
    with pytest.raises(ValueError, match="pointer"):
        segment_matmul(src, torch.tensor([0, 2, 4]), weight)
    with pytest.raises(ValueError, match="1-D"):
        segment_matmul(src, ptr.view(1, 2), weight)


def test_fp8_refuses():
    from ops_gnn import quantize_fp8, segment_matmul_fp8

    src = torch.zeros(4, 160)
    with pytest.raises(RuntimeError, match="CUDA"):
        quantize_fp8(src)
    with pytest.raises(TypeError, match="dtype"):
        quantize_fp8(src.double())
    with pytest.raises(ValueError, match="two dimensions"):
        quantize_fp8(src[0])
    with pytest.raises(ValueError, match="block_rows"):
        quantize_fp8(src, block_rows=64)
    with pytest.raises(TypeError, match="block_rows"):
        quantize_fp8(src, block_rows=True)
    f8 = torch.float8_e4m3fn
    args = [src.to(f8), torch.ones(4, 2), torch.zeros(3, 8, 160).to(f8), torch.ones(3, 1, 2)]
    ptr = torch.tensor([0, 1, 2, 4])
    with pytest.raises(RuntimeError, match="CUDA"):
        segment_matmul_fp8(*args, ptr)
    with pytest.raises(TypeError, match="src dtype"):
        segment_matmul_fp8(src, *args[1:], ptr)
    with pytest.raises(TypeError, match="weight_scale dtype"):
        segment_matmul_fp8(*args[:3], args[3].double(), ptr)
    with pytest.raises(TypeError, match="out_dtype"):
        segment_matmul_fp8(*args, ptr, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="2-D"):
        segment_matmul_fp8(*args)  # three weights and no pointers
    with pytest.raises(ValueError, match="src_scale"):
        segment_matmul_fp8(args[0], torch.ones(4, 1), *args[2:], ptr)
    with pytest.raises(ValueError, match="weight_scale"):
        segment_matmul_fp8(*args[:3], torch.ones(3, 2, 2), ptr)
    with pytest.raises(ValueError, match="pointer"):
        segment_matmul_fp8(*args, ptr[:3])


def test_c_abi_refuses():
    """Bad descriptors and null pointers come back as status codes before anything is launched."""
    from ops_gnn import _cabi

    lib = _cabi.load()
    size = ctypes.c_int64()
    ref = ctypes.byref

    def route(**kw):
        fields = dict(rows=4, experts=16, k=2, groups=1, kept_groups=1, scale=1.0, group_top=1, score=0, renormalize=1,
                      dtype=_cabi.F32)
        fields.update(kw)
        return lib.opsgnn_topk_route(ref(_cabi.RouteDesc(*fields.values())), None, None, None, None, None)

    assert route() == -1 and route(rows=0) == 0
    assert route(groups=3) == -1 and route(k=17) == -1 and route(kept_groups=2) == -1 and route(group_top=3) == -1
    assert route(experts=2048) == -4 and route(experts=64, k=33) == -4 and route(dtype=_cabi.F64) == -2
    assert lib.opsgnn_route_csr_workspace_bytes(10, 4097, ref(size)) == -4
    assert lib.opsgnn_route_csr_workspace_bytes(2 ** 31, 16, ref(size)) == -4
    assert lib.opsgnn_route_csr_workspace_bytes(-1, 16, ref(size)) == -1
    assert lib.opsgnn_route_csr_workspace_bytes(100000, 16, ref(size)) == 0 and size.value > 0
    assert lib.opsgnn_route_csr(1, _cabi.I64, 100000, 16, 1, 1, 1, None, 0, None) == -3

    def matmul(call, *pointers, **kw):
        fields = dict(rows=4, segments=2, width=8, out=8, src_stride=8, weight_segment_stride=64, weight_width_stride=8,
                      weight_out_stride=1, index_type=_cabi.I64, in_type=_cabi.BF16, out_type=_cabi.BF16)
        fields.update(kw)
        return call(ref(_cabi.SegmentMatmulDesc(*fields.values())), *pointers)

    rows, outer, fp8 = lib.opsgnn_segment_matmul, lib.opsgnn_segment_matmul_weight_grad, lib.opsgnn_segment_matmul_fp8
    assert matmul(rows, None, None, None, None, None, 0, None) == -1
    assert matmul(rows, None, None, None, None, None, 0, None, rows=0) == 0
    assert matmul(rows, None, None, None, None, None, 0, None, src_stride=7) == -1
    assert matmul(rows, None, None, None, None, None, 0, None, out_type=_cabi.F32) == -2
    assert matmul(rows, None, None, None, None, None, 0, None, in_type=_cabi.F64, out_type=_cabi.F64) == -2
    assert matmul(rows, None, None, None, None, None, 0, None, index_type=_cabi.F32) == -1
    grads = lib.opsgnn_segment_matmul_grads
    assert matmul(grads, None, None, None, None, 8, None, None, 0, None, 0, None) == -1
    assert matmul(grads, 16, None, None, None, 8, None, None, 0, None, 0, None, rows=0, segments=0) == 0
    assert matmul(grads, 16, 16, 16, 16, 8, 16, 16, 0, None, 0, None, in_type=_cabi.F32, out_type=_cabi.F32, rows=2_000_000) == -3
    assert matmul(lib.opsgnn_segment_matmul_workspace_bytes, 3, ref(size)) == -1
    assert matmul(outer, None, None, None, 8, None, None, 0, None) == -1
    assert matmul(outer, None, None, None, 8, None, None, 0, None, segments=0) == 0
    four = dict(in_type=_cabi.F32, out_type=_cabi.F32, rows=2_000_000)  # large enough to go through bf16 terms
    assert matmul(lib.opsgnn_segment_matmul_workspace_bytes, 0, ref(size), **four) == 0 and size.value >= 6 * (2_000_000 * 8 + 2 * 64)
    assert matmul(rows, 16, 16, 16, 16, None, 0, None, **four) == -3
    assert matmul(lib.opsgnn_segment_matmul_workspace_bytes, 0, ref(size)) == 0 and size.value == 0
    assert matmul(fp8, None, None, None, None, None, None, None) == -2
    assert matmul(fp8, None, None, None, None, None, None, None, in_type=_cabi.F8E4M3) == -1
    assert lib.opsgnn_quantize_fp8(None, _cabi.BF16, 1, 4, 4, 1, None, None, None) == -1
    assert lib.opsgnn_quantize_fp8(None, _cabi.BF16, 1, 0, 4, 1, None, None, None) == 0
    assert lib.opsgnn_quantize_fp8(None, _cabi.BF16, 1, 4, 4, 64, None, None, None) == -1
    assert lib.opsgnn_quantize_fp8(1, _cabi.F64, 1, 4, 4, 1, 1, 1, None) == -2


# ---- topk_route ----------------------------------------------------------------------------------------------------------

ROUTES = [
    # rows, experts, k, score, bias, groups, kept, group_top, renormalize, dtype
    (1, 1, 1, "softmax", False, 1, 1, 2, True, torch.float32),
    (1, 64, 2, "softmax", False, 1, 1, 2, True, torch.bfloat16),
    (37, 7, 3, "sigmoid", False, 1, 1, 2, False, torch.float16),
    (65, 33, 4, "softmax", True, 1, 1, 2, False, torch.float32),
    (129, 100, 8, "softmax", False, 1, 1, 2, False, torch.bfloat16),
    (70, 96, 6, "sigmoid", True, 6, 2, 2, True, torch.float32),
    (70, 96, 6, "softmax", True, 8, 3, 1, True, torch.bfloat16),
    (33, 256, 8, "sigmoid", True, 8, 4, 2, True, torch.float32),
    (33, 256, 8, "sigmoid", False, 8, 4, 1, True, torch.float16),
    (33, 160, 6, "softmax", False, 8, 3, 2, False, torch.float32),
    (9, 384, 8, "sigmoid", True, 1, 1, 2, True, torch.bfloat16),
    (9, 513, 32, "softmax", False, 1, 1, 2, True, torch.float32),
    (5, 1024, 32, "sigmoid", True, 32, 32, 2, True, torch.float32),
    (5, 1024, 9, "softmax", False, 32, 5, 2, True, torch.bfloat16),
    (3, 32, 32, "softmax", False, 1, 1, 2, False, torch.float32),
]


def _route_inputs(case, seed=3):
    rows, experts, k, score, with_bias, groups, kept, top, renormalize, dtype = case
    gen = _gen(seed)
    logits = (torch.randn(rows, experts, generator=gen) * 2).to(dtype)
    bias = torch.randn(experts, generator=gen) * 0.1 if with_bias else None
    return logits, bias


def _check_route(logits, bias, case, weight, index, what):
    rows, experts, k, score, _, groups, kept, top, renormalize, dtype = case
    want_index = _plain_choice(logits, k, score, bias, groups, kept, 1 if groups == 1 else top)
    assert torch.equal(index.cpu(), want_index), what + ": index"
    want = _plain_weight(logits, want_index, score, renormalize, 1.0)
    _within(weight, want, want, experts + 16, what + ": weight")


@requires_gpu
@pytest.mark.parametrize("case", ROUTES, ids=str)
def test_topk_route_forward(cuda_device, case):
    from ops_gnn import topk_route

    logits, bias = _route_inputs(case)
    _, _, k, score, _, groups, kept, top, renormalize, _ = case
    weight, index = topk_route(logits.to(cuda_device), k, score, None if bias is None else bias.to(cuda_device), groups, kept, top,
                               renormalize)
    _check_route(logits, bias, case, weight, index, str(case))


@requires_gpu
@pytest.mark.parametrize("case", [c for c in ROUTES if c[1] >= 32], ids=str)
def test_topk_route_ties_and_masks(cuda_device, case):
    """Whole-number logits (many ties), masked experts, a row with one expert left and a row with none."""
    from ops_gnn import topk_route

    rows, experts, k, score, _, groups, kept, top, renormalize, dtype = case
    logits, bias = _route_inputs(case, 5)
    logits = logits.round()
    logits[torch.rand(logits.shape, generator=_gen(6)) < 0.3] = -math.inf
    logits[0] = -math.inf
    if rows > 2:
        logits[2] = -math.inf
        logits[2, experts // 2] = 1.0
    if rows > 3:
        logits[3] = torch.finfo(dtype).min
    weight, index = topk_route(logits.to(cuda_device), k, score, None if bias is None else bias.to(cuda_device), groups, kept, top,
                               renormalize)
    _check_route(logits, bias, case, weight, index, str(case))
    assert (weight[0] == 0).all()


@requires_gpu
def test_topk_route_nan_and_infinity(cuda_device):
    from ops_gnn import topk_route

    x = torch.randn(6, 40, generator=_gen(1))
    x[1, 3] = math.nan
    x[2, 5] = math.inf
    weight, index = topk_route(x.to(cuda_device), 4)
    plain, plain_index = topk_route(torch.randn(6, 40, generator=_gen(1)).to(cuda_device), 4)
    for r in (0, 3, 4, 5):  # the other rows do not change
        assert torch.equal(weight[r], plain[r]) and torch.equal(index[r], plain_index[r])
    assert torch.isnan(weight[1]).all() and torch.isnan(weight[2]).all()
    assert index[1].tolist() == [0, 1, 2, 3] and index[2].tolist() == [0, 1, 2, 3]
    weight, index = topk_route(x.to(cuda_device), 4, score="sigmoid", renormalize=False)
    assert 3 not in index[1].tolist() and index[2, 0] == 5 and weight[2, 0] == 1 and not torch.isnan(weight).any()


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_topk_route_nan_under_sigmoid(cuda_device, dtype):
    """A NaN comes after every number; where nothing else is left it is chosen and shows as NaN, a masked expert as 0."""
    from ops_gnn import topk_route

    x = torch.full((4, 40), -math.inf, dtype=dtype)
    x[0, 4], x[0, 9], x[0, 30] = 1.0, math.nan, 2.0
    x[1, 2] = math.nan
    x[2] = math.nan
    x[3, 1], x[3, 7] = math.nan, 0.0
    for bias in (None, torch.zeros(40, device=cuda_device)):
        weight, index = topk_route(x.to(cuda_device), 3, score="sigmoid", bias=bias, renormalize=False)
        assert index.tolist() == [[30, 4, 0], [0, 1, 2], [0, 1, 2], [7, 0, 1]]
        nan = [[False, False, False], [False, False, True], [True, True, True], [False, False, True]]
        assert torch.isnan(weight).tolist() == nan
        assert weight[0, 2] == 0 and weight[1, 0] == 0 and weight[3, 1] == 0 and weight[3, 0] == 0.5


@requires_gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,kept", [(1, 1), (8, 3), (10, 4)])
def test_topk_route_many_close_rows(cuda_device, score, groups, kept):
    """Rows whose biased scores come from few logits and few biases: ties by input, and gaps from 1 ulp of fp32 up."""
    from ops_gnn import topk_route

    gen = _gen(51)
    rows, experts, k = 200, 80, 6
    logits = torch.randint(-2, 3, (rows, experts), generator=gen).float() * 0.25
    bias = torch.randint(0, 3, (experts,), generator=gen).float() * 2.0 ** -24 + 0.5
    bias[torch.rand(experts, generator=gen) < 0.3] = 0.75
    weight, index = topk_route(logits.to(cuda_device), k, score, bias.to(cuda_device), groups, kept)
    assert torch.equal(index.cpu(), _plain_choice(logits, k, score, bias, groups, kept, 1 if groups == 1 else 2))


@requires_gpu
def test_topk_route_close_scores(cuda_device):
    """Scores that differ by less than fp32 tells apart: the bias is the only difference, in its last bits."""
    from ops_gnn import topk_route

    experts = 128
    bias = torch.full((experts,), 1.0)
    bias[77] = torch.nextafter(torch.tensor(1.0), torch.tensor(2.0))
    logits = torch.full((3, experts), -20.0)  # sigmoid(-20) = 2e-9: lost beside 1 in fp32
    logits[1, 9] = -19.999
    weight, index = topk_route(logits.to(cuda_device), 3, score="sigmoid", bias=bias.to(cuda_device))
    assert index.tolist() == [[77, 0, 1], [77, 9, 0], [77, 0, 1]]


@requires_gpu
@pytest.mark.parametrize("case", ROUTES, ids=str)
def test_topk_route_gradient(cuda_device, case):
    """Against the formula by float64 autograd of the restated weights, and against central differences of them."""
    from ops_gnn import topk_route

    rows, experts, k, score, _, groups, kept, top, renormalize, dtype = case
    logits, bias = _route_inputs(case)
    if experts > 4:
        logits[rows // 2, 1] = -math.inf
    leaf = logits.to(cuda_device).requires_grad_()
    weight, index = topk_route(leaf, k, score, None if bias is None else bias.to(cuda_device), groups, kept, top, renormalize, 2.5)
    grad = torch.randn(rows, k, generator=_gen(8)).to(dtype)
    got, = torch.autograd.grad(weight, leaf, grad.to(cuda_device))
    assert got.dtype == dtype

    chosen = index.cpu()
    x = logits.double().requires_grad_()
    w = _plain_weight(x, chosen, score, renormalize, 2.5)
    want, = torch.autograd.grad(w, x, grad.double())
    want = torch.nan_to_num(want)  # exp(-inf) in float64 autograd
    s = _plain_scores(logits, score)
    u = 2.5 * grad.double().abs()
    magnitude = torch.zeros_like(s).scatter_add_(1, chosen, u) + (u * s.gather(1, chosen)).sum(1, keepdim=True)
    if renormalize:
        picked = s.gather(1, chosen)
        total = picked.sum(1, keepdim=True)
        mean = (u * picked).sum(1, keepdim=True) / total
        magnitude = torch.zeros_like(s).scatter_add_(1, chosen, (u + mean) / total)
    _within(got, want, magnitude * s, 4 * experts + 64, str(case))

    # Central differences of the restated sum at a few places, step 1e-5: truncation 1e-10, cancellation 1e-11.
    for r, j in ((0, int(chosen[0, 0])), (rows - 1, int(chosen[rows - 1, -1])), (rows // 2, 0)):
        if logits[r, j] == -math.inf:
            continue
        low, high = logits.double(), logits.double()
        low[r, j] -= 1e-5
        high[r, j] += 1e-5
        slope = ((_plain_weight(high, chosen, score, renormalize, 2.5) - _plain_weight(low, chosen, score, renormalize, 2.5))[r]
                 * grad[r].double()).sum() / 2e-5
        bound = 1e-6 + torch.finfo(dtype).eps * abs(float(slope)) + (4 * experts + 64) * STEP * float((magnitude * s)[r, j])
        assert abs(float(slope) - float(got[r, j])) <= bound


@requires_gpu
def test_topk_route_shapes_and_layouts(cuda_device):
    from ops_gnn import topk_route

    x = torch.randn(2, 3, 24, generator=_gen(2)).to(cuda_device)
    weight, index = topk_route(x, 4)
    assert weight.shape == (2, 3, 4) and index.shape == (2, 3, 4) and index.dtype == torch.int64
    flat_weight, flat_index = topk_route(x.view(6, 24), 4)
    assert torch.equal(weight.view(6, 4), flat_weight) and torch.equal(index.view(6, 4), flat_index)
    turned = x.view(6, 24).t().contiguous().t()
    assert torch.equal(topk_route(turned, 4)[1], flat_index)
    shifted = torch.empty(6 * 24 + 1, device=cuda_device)[1:].view(6, 24).copy_(x.view(6, 24))  # 4-byte aligned only
    assert torch.equal(topk_route(shifted, 4)[0], flat_weight)
    one = topk_route(x[0, 0], 4)
    assert torch.equal(one[0], weight[0, 0]) and one[0].shape == (4,)
    empty_weight, empty_index = topk_route(x.new_zeros(0, 24), 4)
    assert empty_weight.shape == (0, 4) and empty_index.shape == (0, 4)
    leaf = x.view(6, 24).clone().requires_grad_()
    weight, index = topk_route(leaf, 4)
    assert weight.requires_grad and not index.requires_grad
    again, = torch.autograd.grad(weight.sum(), leaf)  # weights add up to 1: the gradient of their sum is 0
    assert float(again.abs().max()) <= 8 * STEP


# ---- route_csr -----------------------------------------------------------------------------------------------------------

@requires_gpu
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("count,experts", [(0, 1), (1, 1), (31, 3), (512, 64), (2048, 300), (2049, 8), (5000, 4096), (70001, 257),
                                           (300000, 17)])
def test_route_csr(cuda_device, count, experts, dtype):
    from ops_gnn import route_csr

    gen = _gen(count + experts)
    index = torch.randint(0, experts, (count,), generator=gen, dtype=dtype)
    if count > 40:
        index[torch.rand(count, generator=gen) < 0.1] = experts - 1     # a popular expert
        index[torch.rand(count, generator=gen) < 0.05] = -1             # dropped
        index[7], index[11] = experts, torch.iinfo(dtype).min           # outside the range
    indptr, perm, position = route_csr(index.to(cuda_device), experts)
    label = torch.where((index >= 0) & (index < experts), index, experts).long()
    want = torch.sort(label, stable=True).indices
    assert torch.equal(perm.cpu(), want)
    counts = torch.bincount(label, minlength=experts + 1)[:experts]
    assert torch.equal(indptr.cpu(), torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]))
    back = torch.empty_like(want)
    back[want] = torch.arange(count)
    assert torch.equal(position.cpu(), back)


@requires_gpu
def test_route_csr_shape_and_strides(cuda_device):
    from ops_gnn import route_csr

    index = torch.randint(0, 9, (50, 4), generator=_gen(1)).to(cuda_device)
    indptr, perm, position = route_csr(index, 9)
    assert position.shape == (50, 4) and perm.shape == (200,)
    other = route_csr(index.t().contiguous().t(), 9)
    assert all(torch.equal(a, b) for a, b in zip((indptr, perm, position), other))
    assert torch.equal(index.view(-1)[perm], torch.sort(index.view(-1)).values)


# ---- segment_matmul ------------------------------------------------------------------------------------------------------

MATMULS = [
    # lengths, rows before, rows behind, K, N
    ([5], 0, 0, 16, 24),
    ([1], 0, 0, 8, 8),
    ([3, 0, 1, 130, 0, 64], 0, 0, 64, 96),
    ([0, 0, 0], 0, 7, 32, 16),
    ([127, 128, 129, 1, 0, 255], 3, 5, 136, 264),
    ([40, 30], 2, 0, 7, 5),          # nothing is a whole vector
    ([33, 65, 2], 0, 1, 65, 130),
    ([200, 57], 0, 0, 256, 8),
    ([300], 0, 0, 8, 520),
    ([2] * 70, 0, 0, 72, 40),        # more segments than a warp has lanes
    ([1, 700, 0, 450], 0, 0, 520, 264),
    ([513], 10, 10, 1, 1),
]
KINDS = [torch.bfloat16, torch.float16, torch.float32]


def _matmul_inputs(case, dtype, seed=11):
    lengths, before, behind, k, n = case
    gen = _gen(seed)
    rows = before + sum(lengths) + behind
    src = torch.randn(rows, k, generator=gen).to(dtype)
    weight = torch.randn(len(lengths), k, n, generator=gen).to(dtype)
    grad = torch.randn(rows, n, generator=gen).to(dtype)
    return src, _pointers(lengths, before), weight, grad


@requires_gpu
@pytest.mark.parametrize("dtype", KINDS, ids=str)
@pytest.mark.parametrize("case", MATMULS, ids=str)
def test_segment_matmul(cuda_device, case, dtype):
    """Forward and both gradients, both layouts of the weight, both pointer widths."""
    from ops_gnn import segment_matmul

    src, ptr, weight, grad = _matmul_inputs(case, dtype)
    want = _plain_matmul(src, ptr, weight)
    want_src = _plain_matmul(grad, ptr, weight.transpose(1, 2))
    want_weight = _plain_weight_grad(src, ptr, grad)
    size = _plain_matmul(src.abs(), ptr, weight.abs())
    size_src = _plain_matmul(grad.abs(), ptr, weight.abs().transpose(1, 2))
    size_weight = _plain_weight_grad(src.abs(), ptr, grad.abs())
    longest = max(case[0])
    for turned in (False, True):
        x = src.to(cuda_device).requires_grad_()
        w = (weight.transpose(1, 2).contiguous() if turned else weight).to(cuda_device).requires_grad_()
        pointers = ptr.to(cuda_device).to(torch.int32 if turned else torch.int64)
        out = segment_matmul(x, pointers, w.transpose(1, 2) if turned else w)
        grad_src, grad_weight = torch.autograd.grad(out, (x, w), grad.to(cuda_device))
        if turned:
            grad_weight = grad_weight.transpose(1, 2)
        _within(out, want, size, case[3] + 2, "out")
        _within(grad_src, want_src, size_src, case[4] + 2, "grad_src")
        _within(grad_weight, want_weight, size_weight, longest + 2, "grad_weight")


@requires_gpu
@pytest.mark.parametrize("dtype", KINDS, ids=str)
def test_segment_matmul_layouts(cuda_device, dtype):
    """Rows of a wider matrix, rows at an odd offset, turned rows, a weight of another stride, one weight for all segments."""
    from ops_gnn import segment_matmul

    src, ptr, weight, _ = _matmul_inputs(([30, 0, 140, 9], 1, 2, 64, 72), dtype)
    d_src, d_ptr, d_weight = src.to(cuda_device), ptr.to(cuda_device), weight.to(cuda_device)
    size = _plain_matmul(src.abs(), ptr, weight.abs())
    want = _plain_matmul(src, ptr, weight)
    wide = torch.full((src.size(0), 100), math.nan, dtype=dtype, device=cuda_device)
    for offset in (0, 8, 3):
        view = wide[:, offset:offset + 64]
        view.copy_(d_src)
        _within(segment_matmul(view, d_ptr, d_weight), want, size, 66, f"offset {offset}")
        view.fill_(math.nan)
    _within(segment_matmul(d_src.t().contiguous().t(), d_ptr, d_weight), want, size, 66, "turned rows")
    padded = torch.full((4, 80, 100), math.nan, dtype=dtype, device=cuda_device)
    for k0, n0 in ((0, 0), (8, 16), (1, 3)):
        view = padded[:, k0:k0 + 64, n0:n0 + 72]
        view.copy_(d_weight)
        _within(segment_matmul(d_src, d_ptr, view), want, size, 66, f"weight at {k0}, {n0}")
        view.fill_(math.nan)
    padded = torch.full((4, 80, 104), math.nan, dtype=dtype, device=cuda_device)  # whole vectors, rows apart
    for turned in (False, True):
        view = padded[:, 8:80, 16:80].transpose(1, 2) if turned else padded[:, 8:72, 16:88]
        view.copy_(d_weight)
        _within(segment_matmul(d_src, d_ptr, view), want, size, 66, f"weight of a wider tensor, turned: {turned}")
        view.fill_(math.nan)
    shared = weight[:1].expand(4, -1, -1)
    leaf = weight[:1].to(cuda_device).requires_grad_()
    out = segment_matmul(d_src, d_ptr, leaf.expand(4, -1, -1))
    _within(out, _plain_matmul(src, ptr, shared), _plain_matmul(src.abs(), ptr, shared.abs()), 66, "one weight")
    total, = torch.autograd.grad(out.float().sum(), leaf)
    inside = src[1:180].double()
    # the four segments' gradients are rounded to the dtype each and added in it: four more roundings of the magnitude
    bound = (200 * STEP + 4 * torch.finfo(dtype).eps) * inside.abs().sum(0)
    assert ((total[0].cpu().double() - inside.sum(0).unsqueeze(1)).abs() <= bound.unsqueeze(1)).all()


@requires_gpu
@pytest.mark.parametrize("dtype", KINDS, ids=str)
def test_segment_matmul_empty(cuda_device, dtype):
    from ops_gnn import segment_matmul

    def run(rows, lengths, k, n):
        x = torch.ones(rows, k, dtype=dtype, device=cuda_device, requires_grad=True)
        w = torch.ones(len(lengths), k, n, dtype=dtype, device=cuda_device, requires_grad=True)
        out = segment_matmul(x, _pointers(lengths).to(cuda_device), w)
        return (out,) + torch.autograd.grad(out.sum(), (x, w))

    out, gx, gw = run(5, [], 16, 8)                  # no segments: zeros
    assert out.shape == (5, 8) and not out.any() and not gx.any() and gw.shape == (0, 16, 8)
    out, gx, gw = run(0, [0, 0], 16, 8)              # no rows
    assert out.shape == (0, 8) and gx.shape == (0, 16) and gw.shape == (2, 16, 8) and not gw.any()
    out, gx, gw = run(6, [2, 4], 0, 8)               # empty sums
    assert out.shape == (6, 8) and not out.any() and gx.shape == (6, 0) and gw.shape == (2, 0, 8)
    out, gx, gw = run(6, [2, 4], 16, 0)
    assert out.shape == (6, 0) and not gx.any() and gw.shape == (2, 16, 0)


@requires_gpu
@pytest.mark.parametrize("dtype", KINDS, ids=str)
@pytest.mark.parametrize("k,n", [(64, 128), (200, 72), (33, 5)])
def test_segment_matmul_special_values_stay_in_their_segment(cuda_device, dtype, k, n):
    """NaN and infinities of one segment, and in rows of no segment, reach nothing outside that segment's results."""
    from ops_gnn import segment_matmul

    lengths = [10, 130, 1, 70]
    src, ptr, weight, grad = _matmul_inputs((lengths, 4, 6, k, n), dtype)
    clean = [t.to(cuda_device) for t in (src, ptr, weight, grad)]
    dirty = [t.clone() for t in clean]
    low, high = int(ptr[1]), int(ptr[2])
    for t in (dirty[0], dirty[3]):
        t[low:high] = math.nan
        t[:4] = math.inf
        t[-6:] = -math.inf
    dirty[2][1] = math.inf

    def run(x, p, w, g):
        x, w = x.requires_grad_(), w.requires_grad_()
        out = segment_matmul(x, p, w)
        return (out.detach(),) + torch.autograd.grad(out, (x, w), g)

    plain, other = run(*clean), run(*dirty)
    keep = torch.ones(src.size(0), dtype=torch.bool, device=cuda_device)
    keep[low:high] = False
    for a, b in zip(plain[:2], other[:2]):
        assert torch.equal(a[keep], b[keep]) and torch.isnan(b[low:high]).all()
    for e in (0, 2, 3):
        assert torch.equal(plain[2][e], other[2][e])
    assert torch.isnan(other[2][1]).all()


@requires_gpu
@pytest.mark.parametrize("dtype", KINDS, ids=str)
def test_segment_matmul_infinities_as_the_formula_has_them(cuda_device, dtype):
    from ops_gnn import segment_matmul

    src = torch.ones(140, 64, dtype=dtype)
    weight = torch.ones(1, 64, 72, dtype=dtype) * 0.5
    src[3, 5] = math.inf
    src[4, 5], src[4, 6] = math.inf, -math.inf
    src[139, 0] = -math.inf
    weight[0, 9, 7] = math.inf
    weight[0, :, 8] = 0
    out = segment_matmul(src.to(cuda_device), torch.tensor([0, 140], device=cuda_device), weight.to(cuda_device)).cpu()
    want = src.double() @ weight[0].double()
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out[~torch.isnan(out)].double(), want[~torch.isnan(want)])


@requires_gpu
@pytest.mark.parametrize("dtype", KINDS, ids=str)
def test_segment_matmul_pointers_out_of_range(cuda_device, dtype):
    """Pointers outside the rows count as the nearer end, a segment that ends before it starts is empty."""
    from ops_gnn import segment_matmul

    src, _, weight, grad = _matmul_inputs(([100, 100, 100], 0, 0, 64, 64), dtype)
    ptr = torch.tensor([-5, 40, 2 ** 40, 2 ** 62])
    x, w = src.to(cuda_device).requires_grad_(), weight.to(cuda_device).requires_grad_()
    out = segment_matmul(x, ptr.to(cuda_device), w)
    grad_src, grad_weight = torch.autograd.grad(out, (x, w), grad.to(cuda_device))
    sane = torch.tensor([0, 40, 300, 300])
    _within(out, _plain_matmul(src, sane, weight), _plain_matmul(src.abs(), sane, weight.abs()), 66, "out")
    _within(grad_weight, _plain_weight_grad(src, sane, grad), _plain_weight_grad(src.abs(), sane, grad.abs()), 302, "grad_weight")
    back = segment_matmul(src.to(cuda_device), torch.tensor([0, 200, 100, 300], device=cuda_device), weight.to(cuda_device))
    _within(back[:100], _plain_matmul(src, torch.tensor([0, 200, 200, 300]), weight)[:100],
            _plain_matmul(src.abs(), torch.tensor([0, 200, 200, 300]), weight.abs())[:100], 66, "before the overlap")


@requires_gpu
@pytest.mark.parametrize("dtype", KINDS, ids=str)
def test_segment_matmul_gradients_against_differences(cuda_device, dtype):
    """The sum of out * grad is linear in src and in weight, so differences with a step of 1 are exact up to rounding."""
    from ops_gnn import segment_matmul

    src, ptr, weight, grad = _matmul_inputs(([20, 0, 45], 0, 3, 40, 24), dtype)
    x, w = src.to(cuda_device).requires_grad_(), weight.to(cuda_device).requires_grad_()
    grads = torch.autograd.grad(segment_matmul(x, ptr.to(cuda_device), w), (x, w), grad.to(cuda_device))

    def total(a, b):
        return (_plain_matmul(a, ptr, b) * grad.double()).sum()

    base = total(src, weight)
    for at in ((0, 0), (19, 39), (20, 7), (64, 1), (66, 2)):
        moved = src.double()
        moved[at] += 1
        slope = float(total(moved, weight) - base)
        size = float((grad[at[0]].double().abs() * weight.double().abs().amax(0)[at[1]]).sum())
        assert abs(slope - float(grads[0][at])) <= torch.finfo(dtype).eps * abs(slope) + 26 * STEP * size + 1e-9
    for at in ((0, 0, 0), (1, 3, 4), (2, 39, 23)):
        moved = weight.double()
        moved[at] += 1
        slope = float(total(src, moved) - base)
        size = float((src[:, at[1]].double().abs() * grad[:, at[2]].double().abs()).sum())
        assert abs(slope - float(grads[1][at])) <= torch.finfo(dtype).eps * abs(slope) + 70 * STEP * size + 1e-9


@requires_gpu
def test_segment_matmul_is_reproducible_and_refuses_second_derivatives(cuda_device):
    from ops_gnn import segment_matmul

    src, ptr, weight, grad = [t.to(cuda_device) for t in _matmul_inputs(([500, 3, 900], 0, 0, 256, 256), torch.bfloat16)]
    x, w = src.requires_grad_(), weight.requires_grad_()
    runs = []
    for _ in range(3):
        out = segment_matmul(x, ptr, w)
        runs.append((out.detach(),) + torch.autograd.grad(out, (x, w), grad))
    assert all(torch.equal(a, b) for run in runs[1:] for a, b in zip(runs[0], run))
    out = segment_matmul(x, ptr, w)
    first, = torch.autograd.grad(out.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.float().sum(), w)


# ---- quantize_fp8 --------------------------------------------------------------------------------------------------------

def _plain_quantize(x, block_rows):
    """Block by block on the CPU; torch's own conversion to float8 rounds to nearest even."""
    x = x.double()
    values = torch.empty(x.shape, dtype=torch.float8_e4m3fn)
    rows, width = x.shape
    scale = torch.empty(-(-rows // block_rows), -(-width // 128))
    for i in range(scale.size(0)):
        for j in range(scale.size(1)):
            part = x[i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128]
            finite = part[torch.isfinite(part)].abs()
            top = float(finite.max()) if finite.numel() else 0.0
            p = -126
            while top > 0 and top > 448 * 2.0 ** p:
                p += 1
            s = 2.0 ** p if top > 0 else 1.0
            scale[i, j] = s
            values[i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128] = \
                (part / s).clamp(-448, 448).float().to(torch.float8_e4m3fn)
    return values, scale


@requires_gpu
@pytest.mark.parametrize("dtype", KINDS, ids=str)
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 128), (3, 130), (130, 256), (129, 257), (5, 1000), (260, 24)])
def test_quantize_fp8(cuda_device, rows, width, block_rows, dtype):
    from ops_gnn import quantize_fp8

    gen = _gen(rows * 1000 + width)
    x = torch.randn(rows, width, generator=gen) * torch.exp2(torch.randint(-30, 12, (rows, 1), generator=gen).float())
    x = x.clamp(-60000, 60000).to(dtype)
    if rows > 2:
        x[1] = 0
        x[2, 0] = 448.0
    if width > 128:
        x[0, 5], x[0, 6], x[0, 7] = math.nan, math.inf, -math.inf
    values, scale = quantize_fp8(x.to(cuda_device), block_rows)
    want, want_scale = _plain_quantize(x, block_rows)
    assert torch.equal(scale.cpu(), want_scale)
    assert values.dtype == torch.float8_e4m3fn and values.shape == x.shape
    got, want = values.cpu().float(), want.float()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@requires_gpu
def test_quantize_fp8_extremes_and_borders(cuda_device):
    """The largest and smallest numbers, exact borders of the scale, ties of the rounding, batches, views, no rows."""
    from ops_gnn import quantize_fp8

    big, tiny = torch.finfo(torch.float32).max, torch.finfo(torch.float32).tiny
    x = torch.zeros(8, 128)
    x[0, 0], x[1, 0], x[2, 0], x[3, 0] = big, tiny, 448.0, math.nextafter(448.0, 1000)
    x[3, 0] = float(torch.nextafter(torch.tensor(448.0), torch.tensor(1000.0)))
    x[4, 3] = 2.0 ** -149
    x[5, :3] = torch.tensor([256.0, 17.0, 19.0])     # 17 and 19 lie between 16, 18 and 20: ties to even
    x[6, :2] = torch.tensor([math.inf, math.nan])    # nothing finite: scale 1
    values, scale = quantize_fp8(x.to(cuda_device))
    want, want_scale = _plain_quantize(x, 1)
    assert torch.equal(scale.cpu(), want_scale) and torch.equal(torch.nan_to_num(values.cpu().float()), torch.nan_to_num(want.float()))
    assert scale[2, 0] == 1 and scale[3, 0] == 2 and scale[6, 0] == 1 and scale[7, 0] == 1
    assert values[5, :3].float().tolist() == [256.0, 16.0, 20.0] and values[6, 0].float() == 448

    y = torch.randn(2, 3, 140, 200, generator=_gen(4)).to(cuda_device)
    for block_rows in (1, 128):
        values, scale = quantize_fp8(y, block_rows)
        assert values.shape == y.shape and scale.shape == ((2, 3, 140, 2) if block_rows == 1 else (2, 3, 2, 2))
        one, one_scale = quantize_fp8(y[1, 2], block_rows)
        assert torch.equal(values[1, 2].float(), one.float()) and torch.equal(scale[1, 2], one_scale)
        again, again_scale = quantize_fp8(y.transpose(2, 3).contiguous().transpose(2, 3), block_rows)
        assert torch.equal(values.float(), again.float()) and torch.equal(scale, again_scale)
    values, scale = quantize_fp8(y[:, :, :0])
    assert values.shape == (2, 3, 0, 200) and scale.shape == (2, 3, 0, 2)


# ---- segment_matmul_fp8 --------------------------------------------------------------------------------------------------

def _fp8_inputs(lengths, before, behind, k, n, seed=21, power=False):
    gen = _gen(seed)
    rows = before + sum(lengths) + behind
    src = (torch.randn(rows, k, generator=gen) * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
    weight = (torch.randn(len(lengths), n, k, generator=gen) * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
    blocks, bands = -(-k // 128), -(-n // 128)
    src_scale = torch.rand(rows, blocks, generator=gen) + 0.1
    weight_scale = torch.rand(len(lengths), bands, blocks, generator=gen) + 0.1
    if power:
        src_scale, weight_scale = torch.exp2(torch.round(src_scale * 9 - 5)), torch.exp2(torch.round(weight_scale * 9 - 5))
    return src, src_scale, weight, weight_scale, _pointers(lengths, before)


def _stands_for(values, scale, block_rows):
    v = values.float().double()
    s = scale.double().repeat_interleave(block_rows, -2)[..., :v.size(-2), :].repeat_interleave(128, -1)[..., :v.size(-1)]
    return v * s


FP8S = [
    ([5], 0, 0, 128, 128),
    ([1, 0, 2], 1, 2, 16, 8),
    ([129, 0, 64, 1], 0, 5, 272, 136),
    ([300, 40], 3, 0, 1040, 264),
    ([17, 3], 0, 0, 37, 21),           # nothing is a whole vector
    ([2] * 40, 0, 0, 144, 48),
]


@requires_gpu
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("case", FP8S, ids=str)
def test_segment_matmul_fp8(cuda_device, case, out_dtype):
    from ops_gnn import segment_matmul_fp8

    args = _fp8_inputs(*case, power=out_dtype == torch.float16)
    if out_dtype == torch.float16:  # keep the sums inside the type's range
        args = (args[0], args[1] * 2.0 ** -9, args[2], args[3] * 2.0 ** -9, args[4])
    src, src_scale, weight, weight_scale, ptr = args
    a, b = _stands_for(src, src_scale, 1), _stands_for(weight, weight_scale, 128).transpose(1, 2)
    got = segment_matmul_fp8(*[t.to(cuda_device) for t in args[:4]], ptr.to(cuda_device), out_dtype)
    assert got.dtype == out_dtype
    # K products, one more rounding for each product of two scales and each block's multiply-add
    _within(got, _plain_matmul(a, ptr, b), _plain_matmul(a.abs(), ptr, b.abs()), case[3] + 4, str(case))


@requires_gpu
@pytest.mark.parametrize("m,k,n", [(1, 128, 128), (200, 384, 264), (1, 2048, 16), (130, 48, 1), (0, 128, 128), (5, 0, 9)])
def test_segment_matmul_fp8_dense(cuda_device, m, k, n):
    from ops_gnn import segment_matmul_fp8

    src, src_scale, weight, weight_scale, _ = _fp8_inputs([m], 0, 0, k, n)
    got = segment_matmul_fp8(src.to(cuda_device), src_scale.to(cuda_device), weight[0].to(cuda_device), weight_scale[0].to(cuda_device),
                             out_dtype=torch.float32)
    a, b = _stands_for(src, src_scale, 1), _stands_for(weight, weight_scale, 128)[0]
    assert got.shape == (m, n)
    _within(got, a @ b.t(), a.abs() @ b.abs().t(), k + 4, "dense")


@requires_gpu
def test_segment_matmul_fp8_layouts_and_special_values(cuda_device):
    from ops_gnn import segment_matmul_fp8

    args = _fp8_inputs([70, 0, 130, 4], 0, 3, 256, 128)
    dev = [t.to(cuda_device) for t in args]
    plain = segment_matmul_fp8(*dev, out_dtype=torch.float32)
    assert not plain[-3:].any()
    # Rows of a wider matrix.  Layouts that are not whole 16-byte vectors are summed in another order than the others, so
    # each is held to the bound of its sum, not to the bits of `plain`.
    a, b = _stands_for(args[0], args[1], 1), _stands_for(args[2], args[3], 128).transpose(1, 2)
    want, size = _plain_matmul(a, args[4], b), _plain_matmul(a.abs(), args[4], b.abs())
    for width in (300, 304):
        wide = torch.zeros(207, width, dtype=torch.uint8, device=cuda_device).view(torch.float8_e4m3fn)
        for offset in (0, 16, 5):
            view = wide[:, offset:offset + 256]
            view.view(torch.uint8).copy_(dev[0].view(torch.uint8))
            _within(segment_matmul_fp8(view, *dev[1:], out_dtype=torch.float32), want, size, 260, f"{width}, {offset}")
    turned = dev[2].view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(torch.float8_e4m3fn)
    assert torch.equal(segment_matmul_fp8(dev[0], dev[1].t().contiguous().t(), turned, dev[3], dev[4].int(), torch.float32), plain)
    bits = dev[0].view(torch.uint8).clone()
    bits[70:200, 9] = 0x7f                                     # NaN in one segment
    other = segment_matmul_fp8(bits.view(torch.float8_e4m3fn), *dev[1:], out_dtype=torch.float32)
    assert torch.isnan(other[70:200]).all() and torch.equal(other[:70], plain[:70]) and torch.equal(other[200:], plain[200:])


# ---- together ------------------------------------------------------------------------------------------------------------

def _layer(ops_gnn, x, logits, bias, up, down, k):
    """Rows through their experts: route, dispatch, two products, combine by a CSR product over (row, place) edges."""
    from ops_gnn.torch_sparse_spmm import csr_spmm

    weight, index = ops_gnn.topk_route(logits, k, "sigmoid", bias, groups=4, kept_groups=2)
    indptr, perm, position = ops_gnn.route_csr(index, up.size(0))
    hidden = torch.nn.functional.silu(ops_gnn.segment_matmul(x[perm // k], indptr, up))
    y = ops_gnn.segment_matmul(hidden, indptr, down)
    rows = torch.arange(0, position.numel() + 1, k, device=x.device)
    return csr_spmm(rows, position.view(-1), weight.reshape(-1), y, "sum"), index


@requires_gpu
def test_layer_of_experts(cuda_device):
    """The operators as a layer uses them, forward and backward, against a loop over rows and experts in float64."""
    import ops_gnn

    rows, width, hidden, experts, k = 150, 48, 40, 16, 3
    gen = _gen(31)
    x, logits = torch.randn(rows, width, generator=gen), torch.randn(rows, experts, generator=gen)
    bias = torch.randn(experts, generator=gen) * 0.1
    up = torch.randn(experts, width, hidden, generator=gen) / width ** 0.5
    down = torch.randn(experts, hidden, width, generator=gen) / hidden ** 0.5
    upstream = torch.randn(rows, width, generator=gen)
    leaves = [t.to(cuda_device).requires_grad_() for t in (x, logits, up, down)]
    out, index = _layer(ops_gnn, leaves[0], leaves[1], bias.to(cuda_device), leaves[2], leaves[3], k)
    grads = torch.autograd.grad(out, leaves, upstream.to(cuda_device))

    assert torch.equal(index.cpu(), _plain_choice(logits, k, "sigmoid", bias, 4, 2, 2))
    plain = [t.double().requires_grad_() for t in (x, logits, up, down)]
    weight = _plain_weight(plain[1], index.cpu(), "sigmoid", True, 1.0)
    lines = []
    for r in range(rows):
        parts = [weight[r, j] * (torch.nn.functional.silu(plain[0][r] @ plain[2][e]) @ plain[3][e])
                 for j, e in enumerate(index[r].tolist())]
        lines.append(sum(parts))
    want = torch.stack(lines)
    want_grads = torch.autograd.grad(want, plain, upstream.double())
    # Four stages of fp32 sums of at most 150 terms each, values of order 1: 4 * 150 steps of the largest magnitude
    for got, exact in zip((out,) + grads, (want,) + want_grads):
        bound = 600 * STEP * float(exact.detach().abs().max()) * 4
        assert float((got.detach().cpu().double() - exact.detach()).abs().max()) <= bound


@requires_gpu
def test_layer_in_a_graph_and_on_another_stream(cuda_device):
    """Captured once and replayed with other inputs (other pointers among them), and run on a side stream."""
    import ops_gnn

    rows, width, experts, k = 96, 64, 16, 2
    gen = _gen(41)

    def inputs(seed):
        g = _gen(seed)
        return [torch.randn(rows, width, generator=g).bfloat16().to(cuda_device),
                torch.randn(rows, experts, generator=g).bfloat16().to(cuda_device)]

    up = (torch.randn(experts, width, width, generator=gen) / 8).bfloat16().to(cuda_device)
    quantised = ops_gnn.quantize_fp8(up.transpose(1, 2).contiguous(), 128)

    def run(x, logits):
        weight, index = ops_gnn.topk_route(logits, k)
        indptr, perm, position = ops_gnn.route_csr(index, experts)
        rows_of = x[perm // k]
        y = ops_gnn.segment_matmul(rows_of, indptr, up)
        z = ops_gnn.segment_matmul_fp8(*ops_gnn.quantize_fp8(rows_of), *quantised, indptr)
        return weight, index, indptr, perm, position, y, z

    static = inputs(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = run(*static)
    torch.cuda.current_stream().wait_stream(side)
    plain = run(*static)
    assert all(torch.equal(a, b) for a, b in zip(plain, on_side))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(*static)
    for seed in (2, 3):
        fresh = inputs(seed)
        for buffer, value in zip(static, fresh):
            buffer.copy_(value)
        graph.replay()
        want = run(*fresh)
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), seed
    del graph


@requires_gpu
@pytest.mark.parametrize("dtype", KINDS, ids=str)
@pytest.mark.parametrize("lengths,k,n", [([5000, 0, 70, 1, 3000], 64, 40), ([20000], 8, 136), ([0, 900, 0], 264, 264), ([256, 320, 64], 16, 16)])
def test_segment_matmul_long_sums_in_pieces(cuda_device, dtype, lengths, k, n):
    """Few results and many rows: the weight gradient is summed in pieces of rows and joined, in a fixed order."""
    from ops_gnn import segment_matmul

    src, ptr, weight, grad = _matmul_inputs((lengths, 3, 9, k, n), dtype, 61)
    w = weight.to(cuda_device).requires_grad_()
    args = src.to(cuda_device), ptr.to(cuda_device)
    first, = torch.autograd.grad(segment_matmul(*args, w), w, grad.to(cuda_device))
    again, = torch.autograd.grad(segment_matmul(*args, w), w, grad.to(cuda_device))
    assert torch.equal(first, again)
    _within(first, _plain_weight_grad(src, ptr, grad), _plain_weight_grad(src.abs(), ptr, grad.abs()), max(lengths) + 2, "grad_weight")


@requires_gpu
@pytest.mark.parametrize("dtype", KINDS, ids=str)
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("k,n", [(64, 200), (33, 7)])
def test_segment_matmul_one_gradient_at_a_time(cuda_device, dtype, turned, k, n):
    from ops_gnn import segment_matmul

    src, ptr, weight, grad = [t.to(cuda_device) for t in _matmul_inputs(([90, 0, 300], 1, 2, k, n), dtype)]
    if turned:
        weight = weight.transpose(1, 2).contiguous().transpose(1, 2)
    x, w = src.clone().requires_grad_(), weight.detach().requires_grad_()
    both = torch.autograd.grad(segment_matmul(x, ptr, w), (x, w), grad)
    only_src, = torch.autograd.grad(segment_matmul(x, ptr, weight), x, grad)
    only_weight, = torch.autograd.grad(segment_matmul(src, ptr, w), w, grad)
    assert torch.equal(both[0], only_src) and torch.equal(both[1], only_weight)
    assert both[1].stride() == w.stride()


@requires_gpu
@pytest.mark.parametrize("dtype", KINDS, ids=str)
@pytest.mark.parametrize("rows,k,n,segments", [(3001, 201, 133, 3), (2500, 257, 130, 2), (2100, 130, 641, 1), (9000, 100, 77, 5)])
def test_segment_matmul_large_odd_sizes(cuda_device, dtype, rows, k, n, segments):
    """Sizes that are no whole vectors and large enough for the tensor cores, both layouts of the weight."""
    from ops_gnn import segment_matmul

    lengths = [rows // segments - 7 * e for e in range(segments)]
    src, ptr, weight, grad = _matmul_inputs((lengths, 5, 2, k, n), dtype, 71)
    want, size = _plain_matmul(src, ptr, weight), _plain_matmul(src.abs(), ptr, weight.abs())
    back = weight.transpose(1, 2)
    want_src, size_src = _plain_matmul(grad, ptr, back), _plain_matmul(grad.abs(), ptr, back.abs())
    want_weight, size_weight = _plain_weight_grad(src, ptr, grad), _plain_weight_grad(src.abs(), ptr, grad.abs())
    for turned in (False, True):
        x = src.to(cuda_device).requires_grad_()
        w = (back.contiguous() if turned else weight).to(cuda_device).requires_grad_()
        out = segment_matmul(x, ptr.to(cuda_device), w.transpose(1, 2) if turned else w)
        grad_src, grad_weight = torch.autograd.grad(out, (x, w), grad.to(cuda_device))
        _within(out, want, size, k + 2, "out")
        _within(grad_src, want_src, size_src, n + 2, "grad_src")
        _within(grad_weight.transpose(1, 2) if turned else grad_weight, want_weight, size_weight, max(lengths) + 2, "grad_weight")


@requires_gpu
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("m,k,n", [(700, 304, 333), (513, 1040, 129), (900, 331, 250), (2000, 272, 131)])
def test_segment_matmul_fp8_large_odd_sizes(cuda_device, m, k, n, out_dtype):
    from ops_gnn import segment_matmul_fp8

    args = _fp8_inputs([m // 2, 0, m - m // 2], 0, 0, k, n, 81, True)
    args = (args[0], args[1] * 2.0 ** -9, args[2], args[3] * 2.0 ** -9, args[4])
    a, b = _stands_for(args[0], args[1], 1), _stands_for(args[2], args[3], 128).transpose(1, 2)
    got = segment_matmul_fp8(*[t.to(cuda_device) for t in args], out_dtype)
    _within(got, _plain_matmul(a, args[4], b), _plain_matmul(a.abs(), args[4], b.abs()), k + 4, "fp8")


@requires_gpu
@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp8"])
def test_stalled_wait_raises(cuda_device, kind):
    """Waits without polls give up at once: the launch ends, the next call raises, and the one after it is right again."""
    import ops_gnn

    gen = _gen(91)
    # large enough for every type to run on the kernels that wait (fp32: 2 * 1200 * 256 * 512 = 3.1e8 operations)
    src, weight = torch.randn(1200, 256, generator=gen), torch.randn(2, 256, 512, generator=gen)
    ptr = torch.tensor([0, 500, 1200], device=cuda_device)
    if kind == "fp8":
        operands = ops_gnn.quantize_fp8(src.to(cuda_device)) + ops_gnn.quantize_fp8(weight.transpose(1, 2).contiguous().to(cuda_device), 128)

        def run():
            return ops_gnn.segment_matmul_fp8(*operands, ptr)
    else:
        dtype = torch.bfloat16 if kind == "bf16" else torch.float32
        operands = src.to(dtype).to(cuda_device), ptr, weight.to(dtype).to(cuda_device)

        def run():
            return ops_gnn.segment_matmul(*operands)
    want = run()
    ops_gnn._pybind.device_stall_count(cuda_device.index or 0, True)
    try:
        ops_gnn._pybind.set_wait_polls(0)
        run()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="timed out"):
            run()
    finally:
        ops_gnn._pybind.set_wait_polls(-1)
        ops_gnn._pybind.device_stall_count(cuda_device.index or 0, True)
    assert torch.equal(run(), want)


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("lengths,k,n", [([1], 2048, 256), ([3, 0, 14], 1100, 65), ([130], 4096, 8), ([2, 2], 1536, 1024), ([1], 1025, 72)])
def test_segment_matmul_few_rows_and_long_sums(cuda_device, dtype, lengths, k, n):
    """Serving steps: the sum over the width is cut into pieces and joined; rows of no segment are 0."""
    from ops_gnn import segment_matmul

    src, ptr, weight, grad = _matmul_inputs((lengths, 2, 3, k, n), dtype, 101)
    want, size = _plain_matmul(src, ptr, weight), _plain_matmul(src.abs(), ptr, weight.abs())
    for turned in (False, True):
        x = src.to(cuda_device).requires_grad_()
        w = (weight.transpose(1, 2).contiguous() if turned else weight).to(cuda_device).requires_grad_()
        out = segment_matmul(x, ptr.to(cuda_device), w.transpose(1, 2) if turned else w)
        _within(out, want, size, k + 2, "out")
        assert not out[:2].any() and not out[-3:].any()
        assert torch.equal(out, segment_matmul(x, ptr.to(cuda_device), w.transpose(1, 2) if turned else w))
        grad_src, grad_weight = torch.autograd.grad(out, (x, w), grad.to(cuda_device))
        back = weight.transpose(1, 2)
        _within(grad_src, _plain_matmul(grad, ptr, back), _plain_matmul(grad.abs(), ptr, back.abs()), n + 2, "grad_src")
        _within(grad_weight.transpose(1, 2) if turned else grad_weight, _plain_weight_grad(src, ptr, grad),
                _plain_weight_grad(src.abs(), ptr, grad.abs()), sum(lengths) + 2, "grad_weight")


@requires_gpu
@pytest.mark.parametrize("experts", [5, 40, 300])
def test_topk_route_looks_beyond_ties(cuda_device, experts):
    """The last choice ties with its neighbours by their inputs, and a better expert hides behind them within fp32 rounding."""
    from ops_gnn import topk_route

    logits = torch.full((2, experts), -20.0)
    logits[1, experts - 1] = -19.999  # 2e-12 better beside a bias of 1
    bias = torch.ones(experts, device=cuda_device)
    for k in (1, 2, 3):
        index = topk_route(logits.to(cuda_device), k, score="sigmoid", bias=bias)[1]
        assert index.tolist() == [list(range(k)), [experts - 1] + list(range(k - 1))]


@requires_gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("scale", [1e-30, 1e-3, 1e4, 1e38])
def test_topk_route_fp32_logits_of_any_size(cuda_device, score, scale):
    """The order of fp32 logits is theirs, however close or far apart; one row holds the lowest number as its mask."""
    from ops_gnn import topk_route

    x = torch.randn(50, 200, generator=_gen(111)) * scale
    x[7, ::2] = torch.finfo(torch.float32).min
    x[8] = torch.nextafter(x[8, :1].expand(200), torch.full((200,), math.inf))
    x[8, 150] = x[9, 0]
    x[9, 1:] = x[9, 0] + x[9, 1:] * 1e-7
    _, index = topk_route(x.to(cuda_device), 9, score=score)
    want = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :9]
    if score == "softmax":  # 3.5 sigma times 1e38 is +inf, which makes a softmax NaN: all rank alike, lower numbers first
        want[(x == math.inf).any(1)] = torch.arange(9)
    assert torch.equal(index.cpu(), want)


@requires_gpu
@pytest.mark.parametrize("count,experts", [(70001, 1500), (30000, 2500), (5000003, 40), (9000001, 1200)])
def test_route_csr_many_tiles_and_experts(cuda_device, count, experts):
    from ops_gnn import route_csr

    index = torch.randint(-1, experts, (count,), generator=_gen(count))
    indptr, perm, position = route_csr(index.to(cuda_device), experts)
    label = torch.where(index >= 0, index, experts)
    want = torch.sort(label, stable=True).indices
    assert torch.equal(perm.cpu(), want)
    counts = torch.bincount(label, minlength=experts + 1)[:experts]
    assert torch.equal(indptr.cpu(), torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]))
    back = torch.empty_like(want)
    back[want] = torch.arange(count)
    assert torch.equal(position.cpu(), back)


@requires_gpu
@pytest.mark.parametrize("case", [c for c in ROUTES if c[4]], ids=str)
def test_topk_route_bias_closes_experts(cuda_device, case):
    """A bias of -inf or of the lowest number puts experts behind all others; +inf puts one before them."""
    from ops_gnn import topk_route

    rows, experts, k, score, _, groups, kept, top, renormalize, dtype = case
    logits, bias = _route_inputs(case, 9)
    bias[1::3] = -math.inf
    for special in (None, (4, torch.finfo(torch.float32).min), (experts - 1, math.inf)):
        if special is not None:
            bias[special[0]] = special[1]
        weight, index = topk_route(logits.to(cuda_device), k, score, bias.to(cuda_device), groups, kept, top, renormalize)
        _check_route(logits, bias, case, weight, index, f"{case} {special}")


def _uneven(segments, long, seed):
    """Lengths of many short segments, some empty, with a few long ones between them."""
    lengths = torch.randint(0, 60, (segments,), generator=_gen(seed))
    lengths[torch.rand(segments, generator=_gen(seed + 1)) < 0.2] = 0
    for place, length in long:
        lengths[place] = length
    return lengths.tolist()


@requires_gpu
@pytest.mark.parametrize("dtype", KINDS, ids=str)
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("segments,long,k,n", [(150, [(0, 6000), (1, 700), (149, 2100)], 64, 40), (200, [(70, 9000), (71, 513), (72, 1200)], 17, 130),
                                               (40, [(3, 8000), (9, 3000)], 264, 264), (2000, [(1000, 900), (1999, 4000)], 24, 16)])
def test_segment_matmul_uneven_segments(cuda_device, dtype, turned, segments, long, k, n):
    """Many segments: the weight gradients of the long ones are summed in pieces, those of the others are not."""
    from ops_gnn import segment_matmul

    lengths = _uneven(segments, long, segments)
    src, ptr, weight, grad = _matmul_inputs((lengths, 5, 11, k, n), dtype, 71)
    if turned:
        weight = weight.transpose(1, 2).contiguous().transpose(1, 2)
    x, w = src.to(cuda_device).requires_grad_(), weight.to(cuda_device).requires_grad_()
    grads = torch.autograd.grad(segment_matmul(x, ptr.to(cuda_device), w), (x, w), grad.to(cuda_device))
    back = weight.transpose(1, 2)
    _within(grads[0], _plain_matmul(grad, ptr, back), _plain_matmul(grad.abs(), ptr, back.abs()), n + 2, "grad_src")
    _within(grads[1], _plain_weight_grad(src, ptr, grad), _plain_weight_grad(src.abs(), ptr, grad.abs()), max(lengths) + 2, "grad_weight")


@pytest.mark.parametrize("source", ["segment_matmul_tc.cu", "segment_matmul_promoted.cu"])
def test_kernels_that_give_up_drain_after_the_last_wait(source):
    """A wait may run out in any warp, up to the last one of the block.  So the flag that says so is read behind a barrier that
    follows every wait, and what is in flight (loads, matrix products) ends between it and the release of tensor memory.  When a
    wait runs out in mid flight cannot be arranged from outside, so the order is read from the source."""
    import pathlib

    path = pathlib.Path(__file__).resolve().parent.parent / "ops-gnn_b200" / "csrc" / "cuda" / source
    text = path.read_text()
    last_wait = max(text.rfind("wait.Warp("), text.rfind("wait(&bar"))
    final = text.index("bar.stop != 0")
    release = text.index("TmemFree(", final)
    assert last_wait < final and "__syncthreads();" in text[last_wait:final]
    for drained in ("BarTry(&bar.full", "tc::Commit(&bar.drain)", "BarTry(&bar.drain"):
        at = text.index(drained, final)
        assert at < release and text.count(drained) == 1
        assert "__syncthreads();" in text[at:release]


@requires_gpu
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_waits_of_a_single_poll(cuda_device, kind):
    """One poll for each wait: the launch ends, complete or given up anywhere within; either way the next one is right."""
    import ops_gnn

    gen = _gen(93)
    dtype = torch.bfloat16 if kind == "bf16" else torch.float32
    src = torch.randn(3000, 512, generator=gen).to(dtype).to(cuda_device).requires_grad_()
    weight = torch.randn(3, 512, 512, generator=gen).to(dtype).to(cuda_device).requires_grad_()
    grad = torch.randn(3000, 512, generator=gen).to(dtype).to(cuda_device)
    ptr = torch.tensor([0, 700, 701, 3000], device=cuda_device)

    def run():
        out = ops_gnn.segment_matmul(src, ptr, weight)
        return (out.detach(),) + torch.autograd.grad(out, (src, weight), grad)

    want = run()
    device = cuda_device.index or 0
    try:
        ops_gnn._pybind.set_wait_polls(1)
        for _ in range(3):
            ops_gnn._pybind.device_stall_count(device, True)
            ops_gnn._pybind.segment_matmul_forward(src.detach(), ptr, weight.detach())
            torch.cuda.synchronize()
    finally:
        ops_gnn._pybind.set_wait_polls(-1)
        ops_gnn._pybind.device_stall_count(device, True)
    assert all(torch.equal(a, b) for a, b in zip(run(), want))


def _matches(actual, product, a, b, terms, what):
    """product(a, b) in 64 bits: NaN and infinities where it has them when rounded to the type, finite results within the bound of
    _within.

    Left out: results whose finite terms' magnitudes add up to 2^127 or more, unless all terms are finite and have one sign.  A sum
    in fp32 of some of the terms may pass 2^128, as an infinity of either sign, before the others bring the total back or an
    infinity of the other sign joins it, so such a result depends on the order of the sum.  Terms of one sign only grow, and smaller
    magnitudes never get there, in any order."""
    expected, magnitude = product(a, b), product(a.abs(), b.abs())
    a0, b0 = [torch.where(torch.isfinite(t), t, torch.zeros_like(t)) for t in (a, b)]
    size = product(a0.abs(), b0.abs())
    open_ = (size >= 2.0 ** 127) & ~(torch.isfinite(magnitude) & (expected.abs() >= magnitude * (1 - 1e-12)))
    got, want = actual.detach().cpu(), expected.to(actual.dtype)
    assert not open_.all()
    got, want, expected, magnitude = [t[~open_] for t in (got, want, expected, magnitude)]
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what + ": NaN"
    assert torch.equal(got[torch.isinf(got)], want[torch.isinf(got)]) and torch.equal(torch.isinf(got), torch.isinf(want)), what + ": infinities"
    fine = torch.isfinite(want)
    _within(got[fine], expected[fine], magnitude[fine], terms, what)


@requires_gpu
@pytest.mark.parametrize("kind", ["nan", "infinite", "above bf16", "overflow"])
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("lengths,k,n", [([700, 0, 1000, 403], 264, 200), ([6000, 30, 4500], 72, 264), ([5000, 4000], 40, 520), ([3, 2500], 130, 264)])
def test_segment_matmul_special_values_in_fp32_terms(cuda_device, lengths, k, n, turned, kind):
    """fp32 products large enough for the sums of bf16 terms (2e8 operations, 2048 rows for gradients), in one piece and in
    pieces: NaN, infinities, numbers that round to an infinity in bf16 and sums that overflow."""
    from ops_gnn import segment_matmul

    assert 2 * sum(lengths) * k * n >= 1.5e8 and sum(lengths) >= 2048
    src, ptr, weight, grad = _matmul_inputs((lengths, 3, 5, k, n), torch.float32, 121)
    last, middle = sum(lengths) + 2, 3 + lengths[0] // 2  # the last row of the last segment, one within the first
    if kind == "nan":
        src[last, 3], grad[middle, n - 1] = math.nan, math.nan
    elif kind == "infinite":
        src[last, 3], src[middle, 5], grad[middle, n - 1] = math.inf, -math.inf, math.inf
        weight[0, 5, 2], weight[-1, 7, 9] = 0.0, math.inf
        src[middle + 1, 5] = math.inf  # and minus infinity in the same column: NaN in its weight gradient
    elif kind == "above bf16":  # times small numbers only
        src[last, 3], weight[-1, 3], grad[last] = 3.398e38, weight[-1, 3] * 1e-30, grad[last] * 1e-30
        grad[middle, 4], weight[0, :, 4], src[middle] = -3.398e38, weight[0, :, 4] * 1e-30, src[middle] * 1e-30
    else:
        src[last], weight[-1], grad[middle] = 1e38, weight[-1].abs() * 1e38, 2e38
        src[middle] = src[middle].abs() + 1
    back = weight.transpose(1, 2)
    x = src.to(cuda_device).requires_grad_()
    w = (back.contiguous() if turned else weight).to(cuda_device).requires_grad_()
    out = segment_matmul(x, ptr.to(cuda_device), w.transpose(1, 2) if turned else w)
    grad_src, grad_weight = torch.autograd.grad(out, (x, w), grad.to(cuda_device))
    _matches(out, lambda a, b: _plain_matmul(a, ptr, b), src, weight, k + 2, "out")
    _matches(grad_src, lambda a, b: _plain_matmul(a, ptr, b), grad, back, n + 2, "grad_src")
    _matches(grad_weight.transpose(1, 2) if turned else grad_weight, lambda a, b: _plain_weight_grad(a, ptr, b), src, grad,
             max(lengths) + 2, "grad_weight")


@requires_gpu
def test_segment_matmul_fp32_with_a_row_of_nan_takes_no_longer(cuda_device):
    """One row of NaN makes a whole weight gradient NaN; nothing is summed again for it."""
    from ops_gnn import segment_matmul

    src, ptr, weight, grad = [t.to(cuda_device) for t in _matmul_inputs(([2000, 6000, 192], 0, 0, 512, 512), torch.float32, 131)]
    dirty = src.clone()
    dirty[-200] = math.nan

    def step(values):
        x, w = values.requires_grad_(), weight.requires_grad_()
        times = []
        for _ in range(8):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            out = segment_matmul(x, ptr, w)
            grads = torch.autograd.grad(out, (x, w), grad)
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end))
        return min(times[2:]), grads[1]

    clean, _ = step(src)
    slow, grad_weight = step(dirty)
    assert torch.isnan(grad_weight[1]).all() and torch.isfinite(grad_weight[0]).all() and torch.isfinite(grad_weight[2]).all()
    assert slow <= 2 * clean, (slow, clean)


def test_teams_sum_outside_of_branches():
    """Sums over a team of lanes are warp-wide shuffles: a condition in front of one that differs from row to row keeps lanes away
    from it.  So none stands behind the ? of a condition, but for those of the call's own choices, alike in all rows."""
    import pathlib
    import re

    source = pathlib.Path(__file__).resolve().parent.parent / "ops-gnn_b200" / "csrc" / "cuda" / "route.cu"
    guarded = re.findall(r"([\w.:]+(?: (?:==|!=|<=|>=|<|>) [\w.]+)?) \?[^;]*?(?:Team|Warp)(?:Sum|Max)", source.read_text())
    assert set(guarded) <= {"p.renormalize", "p.softmax"}, guarded


@requires_gpu
@pytest.mark.parametrize("dtype", KINDS, ids=str)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("experts,k", [(40, 4), (33, 3), (200, 8), (96, 12), (1000, 2)])
def test_topk_route_gradient_beside_masked_rows(cuda_device, dtype, score, renormalize, experts, k):
    """Rows that the mask leaves nothing of have no gradient, and their neighbours keep theirs to the bit."""
    from ops_gnn import topk_route

    x = (torch.randn(23, experts, generator=_gen(151)) * 2).to(dtype)
    grad = torch.randn(23, k, generator=_gen(152)).to(dtype).to(cuda_device)
    plain = x.to(cuda_device).requires_grad_()
    want, = torch.autograd.grad(topk_route(plain, k, score, renormalize=renormalize)[0], plain, grad)
    masked = [0, 2, 5, 6, 15, 22]
    x[masked] = -math.inf
    leaf = x.to(cuda_device).requires_grad_()
    weight, _ = topk_route(leaf, k, score, renormalize=renormalize)
    got, = torch.autograd.grad(weight, leaf, grad)
    want[masked] = 0
    assert not weight[masked].any() and torch.equal(got, want)


@requires_gpu
@pytest.mark.parametrize("experts,k", [(16, 2), (40, 12)])
def test_topk_route_gradient_of_tiny_scores(cuda_device, experts, k):
    """Sigmoid scores near the smallest number of fp32, whose sum no gradient can be divided by: their shares of it are ordinary.

    A score of 3e-39 has steps of 2^-149, 4.7e-7 of its value or 4 * 2^-23: three of them (score, sum, share) make 12 steps more
    than the bound of ordinary scores counts."""
    from ops_gnn import topk_route

    gen = _gen(161)
    x = -88.2 + 0.4 * torch.rand(30, experts, generator=gen)
    x[7] = -math.inf
    grad = torch.randn(30, k, generator=gen) * 20
    leaf = x.to(cuda_device).requires_grad_()
    weight, index = topk_route(leaf, k, "sigmoid")
    got, = torch.autograd.grad(weight, leaf, grad.to(cuda_device))
    chosen = index.cpu()
    s = torch.sigmoid(x.double())
    picked = s.gather(1, chosen)
    share = picked / picked.sum(1, keepdim=True).clamp(min=1e-300)
    u = grad.double()
    want = torch.zeros_like(s).scatter_(1, chosen, share * (1 - picked) * (u - (u * share).sum(1, keepdim=True)))
    size = torch.zeros_like(s).scatter_(1, chosen, share * (u.abs() + (u.abs() * share).sum(1, keepdim=True)))
    _within(got, want, size, 4 * experts + 64 + 12, "gradient")
    _within(weight, share, share, experts + 16 + 12, "weight")


@requires_gpu
@pytest.mark.parametrize("dtype", KINDS, ids=str)
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("experts,k", [(40, 4), (33, 3), (200, 8), (256, 12), (1000, 2)])
def test_topk_route_gradient_of_a_row_without_a_softmax(cuda_device, dtype, renormalize, experts, k):
    """A NaN or +inf anywhere in a row makes its softmax NaN: the weights, and the gradient of every logit.  Other rows keep theirs."""
    from ops_gnn import _pybind, topk_route

    x = (torch.randn(9, experts, generator=_gen(141)) * 2).to(dtype)
    grad = torch.randn(9, k, generator=_gen(142)).to(dtype).to(cuda_device)
    plain = x.to(cuda_device).requires_grad_()
    want, = torch.autograd.grad(topk_route(plain, k, renormalize=renormalize)[0], plain, grad)
    low = x.argmin(1)  # not among the chosen
    x[1, low[1]], x[3, low[3]], x[6, 0] = math.nan, math.inf, math.nan
    x[6, 1] = -math.inf
    leaf = x.to(cuda_device).requires_grad_()
    weight, index = topk_route(leaf, k, renormalize=renormalize)
    got, = torch.autograd.grad(weight, leaf, grad)
    for r in range(9):
        if r in (1, 3, 6):
            assert torch.isnan(weight[r]).all() and torch.isnan(got[r]).all(), r
        else:
            assert torch.equal(got[r], want[r]), r
    # without the forward pass's note of such rows
    alone = _pybind.topk_route_backward(leaf.detach(), index, grad, 0, renormalize, 1.0)
    assert torch.equal(torch.isnan(alone), torch.isnan(got)) and torch.equal(torch.nan_to_num(alone), torch.nan_to_num(got))


def _waits(run, device):
    """Whether a call runs on the kernels that wait for their loads (the tensor cores'): without polls these report a stall."""
    from ops_gnn import _pybind

    index = device.index or 0
    torch.cuda.synchronize()
    _pybind.device_stall_count(index, True)
    try:
        _pybind.set_wait_polls(0)
        run()
        torch.cuda.synchronize()
        return _pybind.device_stall_count(index, True) > 0
    finally:
        _pybind.set_wait_polls(-1)
        _pybind.device_stall_count(index, True)


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("rows,k,n,segments", [(2100, 130, 641, 1), (3000, 257, 131, 1), (1, 2049, 25000, 1), (2100, 130, 641, 3), (2000, 25001, 1, 1)])
def test_segment_matmul_odd_sizes_reach_the_tensor_cores(cuda_device, dtype, turned, rows, k, n, segments):
    """Large products of odd sizes run on the tensor cores, also where a dimension has one element: nothing steps over its stride."""
    from ops_gnn import segment_matmul

    lengths = [rows] if segments == 1 else [rows - 1200, 0, 1200]
    src, ptr, weight, grad = _matmul_inputs((lengths, 0, 0, k, n), dtype, 171)
    back = weight.transpose(1, 2)
    x, p, g = src.to(cuda_device).requires_grad_(), ptr.to(cuda_device), grad.to(cuda_device)
    w = (back.contiguous() if turned else weight).to(cuda_device)
    call = (lambda a: segment_matmul(a, p, w.transpose(1, 2) if turned else w))
    out = call(x)
    grad_src, = torch.autograd.grad(out, x, g)
    _within(out, _plain_matmul(src, ptr, weight), _plain_matmul(src.abs(), ptr, weight.abs()), k + 2, "out")
    _within(grad_src, _plain_matmul(grad, ptr, back), _plain_matmul(grad.abs(), ptr, back.abs()), n + 2, "grad_src")
    assert _waits(lambda: call(x.detach()), cuda_device), "forward"
    out = call(x)
    assert _waits(lambda: torch.autograd.grad(out, x, g), cuda_device), "grad_src"


@requires_gpu
@pytest.mark.parametrize("m,k,n", [(1, 2049, 25000), (700, 331, 333), (2000, 25001, 1)])
def test_segment_matmul_fp8_odd_sizes_reach_the_tensor_cores(cuda_device, m, k, n):
    from ops_gnn import segment_matmul_fp8

    src, src_scale, weight, weight_scale, ptr = [t.to(cuda_device) for t in _fp8_inputs([m], 0, 0, k, n, 181)]
    for call in (lambda: segment_matmul_fp8(src, src_scale, weight, weight_scale, ptr, torch.float32),
                 lambda: segment_matmul_fp8(src, src_scale, weight[0], weight_scale[0], out_dtype=torch.float32)):
        a, b = _stands_for(src.cpu(), src_scale.cpu(), 1), _stands_for(weight.cpu(), weight_scale.cpu(), 128)[0]
        _within(call(), a @ b.t(), a.abs() @ b.abs().t(), k + 4, "fp8")
        assert _waits(call, cuda_device)


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("lengths,k,n", [([9001], 15, 15), ([300], 33, 33), ([700, 0, 1400], 7, 21), ([3] * 400 + [17000], 15, 9)])
def test_segment_matmul_weight_gradient_of_long_narrow_segments(cuda_device, dtype, lengths, k, n):
    """Few columns, none of them whole vectors, and long segments: the weight gradient does not run as one block's sum per segment,
    alone or together with the gradient of src."""
    from ops_gnn import segment_matmul

    src, ptr, weight, grad = _matmul_inputs((lengths, 1, 2, k, n), dtype, 191)
    x, w = src.to(cuda_device).requires_grad_(), weight.to(cuda_device).requires_grad_()
    p, g = ptr.to(cuda_device), grad.to(cuda_device)
    want, size = _plain_weight_grad(src, ptr, grad), _plain_weight_grad(src.abs(), ptr, grad.abs())
    only, = torch.autograd.grad(segment_matmul(x.detach(), p, w), w, g)
    grad_src, both = torch.autograd.grad(segment_matmul(x, p, w), (x, w), g)
    _within(only, want, size, max(lengths) + 2, "grad_weight")
    assert torch.equal(only, both)
    back = weight.transpose(1, 2)
    _within(grad_src, _plain_matmul(grad, ptr, back), _plain_matmul(grad.abs(), ptr, back.abs()), n + 2, "grad_src")
    for leaves in ((w,), (x, w)):
        out = segment_matmul(x if len(leaves) == 2 else x.detach(), p, w)
        assert _waits(lambda: torch.autograd.grad(out, leaves, g), cuda_device)


def test_weight_gradients_of_very_many_segments_are_not_cut():
    """Where a piece goes is told by twice its segment's number and one, in 32 bits."""
    from ops_gnn import _cabi

    lib, size = _cabi.load(), ctypes.c_int64()
    for kind in (_cabi.BF16, _cabi.F16):
        for segments, cut in ((1000, True), (2 ** 30 - 1, True), (2 ** 30, False), (2 ** 31 - 600, False)):
            desc = _cabi.SegmentMatmulDesc(2 ** 20, segments, 8, 8, 8, 64, 8, 1, _cabi.I64, kind, kind)
            assert lib.opsgnn_segment_matmul_workspace_bytes(ctypes.byref(desc), 1, ctypes.byref(size)) == 0
            assert (size.value > 0) == cut


@requires_gpu
@pytest.mark.parametrize("dtype", KINDS, ids=str)
@pytest.mark.parametrize("lengths,k,n", [([9000, 0, 70, 1, 300, 3000], 64, 40), ([4000, 300, 0, 1, 4001, 2], 264, 264), ([8192], 16, 16), ([0, 8500, 0], 128, 24),
                                         ([600] * 15, 8, 136)])
def test_segment_matmul_few_results_of_many_rows_in_pieces(cuda_device, dtype, lengths, k, n):
    """Weight gradients of fewer tiles than SMs: pieces of long segments, empty and one-row segments between them, and segments
    that end and start within one piece's length of rows, which is what two slots for each are for."""
    from ops_gnn import _cabi, segment_matmul

    src, ptr, weight, grad = _matmul_inputs((lengths, 3, 9, k, n), dtype, 201)
    if dtype != torch.float32:
        size, kind = ctypes.c_int64(), _cabi.BF16 if dtype == torch.bfloat16 else _cabi.F16
        desc = _cabi.SegmentMatmulDesc(src.size(0), len(lengths), k, n, k, k * n, n, 1, _cabi.I64, kind, kind)
        assert _cabi.load().opsgnn_segment_matmul_workspace_bytes(ctypes.byref(desc), 1, ctypes.byref(size)) == 0
        assert size.value > 0, "not in pieces any more: longer segments, please"
    w = weight.to(cuda_device).requires_grad_()
    x = src.to(cuda_device)
    p, g = ptr.to(cuda_device), grad.to(cuda_device)
    first, = torch.autograd.grad(segment_matmul(x, p, w), w, g)
    again, = torch.autograd.grad(segment_matmul(x, p, w), w, g)
    assert torch.equal(first, again)
    _within(first, _plain_weight_grad(src, ptr, grad), _plain_weight_grad(src.abs(), ptr, grad.abs()), max(lengths) + 2, "grad_weight")
    turned = weight.transpose(1, 2).contiguous().to(cuda_device).requires_grad_()
    other, = torch.autograd.grad(segment_matmul(x, p, turned.transpose(1, 2)), turned, g)
    _within(other.transpose(1, 2), _plain_weight_grad(src, ptr, grad), _plain_weight_grad(src.abs(), ptr, grad.abs()), max(lengths) + 2, "turned")


@requires_gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,kept,top", [(1, 1, 2), (8, 3, 2), (8, 4, 1)])
@pytest.mark.parametrize("mask", [-1e4, -1e9, torch.finfo(torch.float32).min, 1e6])
def test_topk_route_biases_of_any_size(cuda_device, score, groups, kept, top, mask):
    """Some biases as large as masks are, the others so close that fp32 does not tell their sums with the scores apart."""
    from ops_gnn import topk_route

    gen = _gen(211)
    rows, experts, k = 150, 80, 6
    logits = torch.randint(-2, 3, (rows, experts), generator=gen).float() * 0.25
    bias = torch.randint(0, 3, (experts,), generator=gen).float() * 2.0 ** -24 + 0.5
    for few in (slice(1, None, 5), slice(20, 30)):  # some of each group, one whole group of eight
        some = bias.clone()
        some[few] = mask
        weight, index = topk_route(logits.to(cuda_device), k, score, some.to(cuda_device), groups, kept, top)
        assert torch.equal(index.cpu(), _plain_choice(logits, k, score, some, groups, kept, 1 if groups == 1 else top))


@requires_gpu
@pytest.mark.parametrize("groups,kept", [(1, 1), (8, 4)])
def test_topk_route_with_a_finite_mask_in_the_bias_takes_no_longer(cuda_device, groups, kept):
    """The error of a masked expert's score is as large as its mask, and has no part in choosing among the others."""
    from ops_gnn import topk_route

    gen = torch.Generator(device=cuda_device).manual_seed(221)
    logits = torch.randn(65536, 256, generator=gen, device=cuda_device)
    bias = torch.randn(256, generator=gen, device=cuda_device) * 0.05
    masked = bias.clone()
    masked[::5] = -1e9

    def best(b):
        times = []
        for _ in range(8):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            for _ in range(8):
                topk_route(logits, 8, "sigmoid", b, groups, kept)
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end))
        return min(times[2:])

    plain, other = best(bias), best(masked)
    assert other <= 1.5 * plain, (other, plain)


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("lengths,k,n", [([9000], 16, 15), ([300, 500], 15, 16), ([600], 264, 15), ([3000, 17000], 7, 24)])
def test_segment_matmul_gradients_alone_and_together(cuda_device, dtype, turned, lengths, k, n):
    """The gradient of src has the same bits alone and beside the weight's, also where only the latter's operands are copied."""
    from ops_gnn import segment_matmul

    src, ptr, weight, grad = [t.to(cuda_device) for t in _matmul_inputs((lengths, 1, 2, k, n), dtype, 231)]
    if turned:
        weight = weight.transpose(1, 2).contiguous().transpose(1, 2)
    x, w = src.clone().requires_grad_(), weight.detach().requires_grad_()
    both = torch.autograd.grad(segment_matmul(x, ptr, w), (x, w), grad)
    only_src, = torch.autograd.grad(segment_matmul(x, ptr, weight), x, grad)
    only_weight, = torch.autograd.grad(segment_matmul(src, ptr, w), w, grad)
    assert torch.equal(both[0], only_src) and torch.equal(both[1], only_weight)
    assert both[1].stride() == w.stride()


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_training_step_in_a_graph(cuda_device, dtype):
    """Choice, dispatch, products and all gradients, captured once and replayed on other inputs: the bits of eager passes."""
    import ops_gnn

    tokens, width, hidden, experts, k = 1100, 64, 72, 12, 2
    gen = _gen(241)
    weight = (torch.randn(experts, width, hidden, generator=gen) / 8).to(dtype).to(cuda_device)

    def inputs(seed):
        g = _gen(seed)
        logits = torch.randn(tokens, experts, generator=g)
        logits[5] = -math.inf
        return [torch.randn(tokens, width, generator=g).to(dtype).to(cuda_device), logits.to(dtype).to(cuda_device),
                torch.randn(tokens, hidden, generator=g).to(dtype).to(cuda_device)]

    def step(x, logits, upstream):
        leaves = [t.detach().requires_grad_() for t in (x, logits, weight)]
        chosen, index = ops_gnn.topk_route(leaves[1], k)
        indptr, perm, position = ops_gnn.route_csr(index, experts)
        y = ops_gnn.segment_matmul(leaves[0][perm // k], indptr, leaves[2])
        out = (y[position.view(-1)].view(tokens, k, hidden) * chosen.unsqueeze(-1)).sum(1)
        return (out.detach(),) + torch.autograd.grad(out, leaves[1:], upstream)

    static = inputs(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(*static)
    for seed in (2, 3):
        fresh = inputs(seed)
        for buffer, value in zip(static, fresh):
            buffer.copy_(value)
        graph.replay()
        want = step(*fresh)
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), seed
    del graph


@requires_gpu
@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp8"])
def test_products_past_32_bit_offsets(cuda_device, kind):
    """More than 2^31 values in src and in the result, the last segment past both: rows at the ends and at the 2^31st value."""
    import ops_gnn

    rows, k, n, segments = 4_200_000, 520, 520, 3
    assert rows * k > 2 ** 31
    if torch.cuda.get_device_properties(cuda_device).total_memory < 120 * 2 ** 30:
        pytest.skip("needs a GPU of 120 GiB")
    gen = torch.Generator(device=cuda_device).manual_seed(251)
    dtype = torch.float32 if kind == "fp32" else torch.bfloat16
    src = torch.empty(rows, k, dtype=dtype, device=cuda_device)
    for part in src.split(500_000):
        part.normal_(generator=gen)
    weight = torch.randn(segments, k, n, generator=gen, device=cuda_device).to(dtype)
    ptr = torch.tensor([0, 4_000_000, 4_199_000, rows - 1], device=cuda_device)
    edge = 2 ** 31 // k
    look = torch.tensor([0, 1, edge - 1, edge, edge + 1, 3_999_999, 4_000_000, 4_198_999, 4_199_000, rows - 2], device=cuda_device)
    which = torch.bucketize(look, ptr[1:], right=True)
    if kind == "fp8":
        values, scale = ops_gnn.quantize_fp8(src)
        w8, w8_scale = ops_gnn.quantize_fp8(weight.transpose(1, 2).contiguous(), 128)
        out = ops_gnn.segment_matmul_fp8(values, scale, w8, w8_scale, ptr)
        part, part_scale = ops_gnn.quantize_fp8(src[look])
        assert torch.equal(part.view(torch.uint8), values.view(torch.uint8)[look]) and torch.equal(part_scale, scale[look])
        a, b = _stands_for(part.cpu(), part_scale.cpu(), 1), _stands_for(w8.cpu(), w8_scale.cpu(), 128).transpose(1, 2)
    else:
        out = ops_gnn.segment_matmul(src, ptr, weight)
        a, b = src[look].cpu().double(), weight.cpu().double()
    want = torch.stack([a[i] @ b[int(e)] for i, e in enumerate(which)])
    size = torch.stack([a[i].abs() @ b[int(e)].abs() for i, e in enumerate(which)])
    _within(out[look], want, size, k + 4, "out")
    assert not out[-1].any()
    if kind == "fp8":
        return
    # The weight gradient of the last segment, which lies past the 2^31st value of both.
    grad_weight = ops_gnn._pybind.segment_matmul_weight_grad(src, ptr, out)
    x, g = src[4_199_000:rows - 1].cpu(), out[4_199_000:rows - 1].cpu()
    last = torch.tensor([0, x.size(0)])
    _within(grad_weight[2:], _plain_weight_grad(x, last, g), _plain_weight_grad(x.abs(), last, g.abs()), x.size(0) + 2, "grad_weight")


@requires_gpu
def test_topk_route_past_32_bit_offsets(cuda_device):
    from ops_gnn import topk_route

    rows, experts = 2_100_001, 1024
    assert rows * experts > 2 ** 31
    gen = torch.Generator(device=cuda_device).manual_seed(261)
    logits = torch.empty(rows, experts, dtype=torch.bfloat16, device=cuda_device)
    for part in logits.split(300_000):
        part.normal_(generator=gen)
    leaf = logits.requires_grad_()
    weight, index = topk_route(leaf, 4)
    grad, = torch.autograd.grad(weight, leaf, weight.detach())
    tail = logits.detach()[-3:].clone().requires_grad_()
    tail_weight, tail_index = topk_route(tail, 4)
    tail_grad, = torch.autograd.grad(tail_weight, tail, tail_weight.detach())
    assert torch.equal(weight[-3:], tail_weight) and torch.equal(index[-3:], tail_index) and torch.equal(grad[-3:], tail_grad)
    assert torch.equal(index[-3:].cpu(), _plain_choice(tail.detach().cpu(), 4, "softmax", None, 1, 1, 1))
