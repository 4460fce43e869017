"""Expert products of MXFP4 operands against 64-bit sums of the values they stand for, on the B200.

Tolerance: products of two codes and two powers of two are exact; the FP32 sum of C of them in
any order and grouping stays within C * 2^-22 of the sum of magnitudes (cut, not rounded, at each
step and when a group of products is aligned), and the output is rounded once to its type.
"""

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA device required"),
]

from loraforge_b200 import _native  # noqa: E402
from loraforge_b200.ops.experts import combine_experts, route_experts  # noqa: E402
from loraforge_b200.ops.mxfp4 import (  # noqa: E402
    MxTensor, expert_linear_mxfp4, mxfp4_dequantize, mxfp4_quantize)

UNIT = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def random_mx(g, *shape, low=-3, high=3):
    """Every code and a spread of scales, as bytes."""
    codes = torch.randint(0, 256, (*shape[:-1], shape[-1] // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.randint(127 + low, 128 + high, (*shape[:-1], shape[-1] // 32), generator=g, device="cuda")
    return MxTensor(codes, scales.to(torch.uint8))


def values64(q):
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float64, device="cuda")
    v = table[torch.stack((q.codes & 15, q.codes >> 4), -1).flatten(-2).long()].unflatten(-1, (-1, 32))
    powers = torch.tensor([math.ldexp(1.0, i - 127) for i in range(255)] + [math.nan], dtype=torch.float64, device="cuda")
    return (v * powers[q.scales.long()][..., None]).flatten(-2)


def make(counts, N, K, seed, tail=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    R = sum(counts) + tail
    tokens = max(1, R // 2)
    offsets = torch.tensor([0, *counts], device="cuda").cumsum(0).to(torch.int32)
    rows = torch.randint(0, tokens, (R,), generator=g, device="cuda").to(torch.int32)
    return random_mx(g, tokens, K), random_mx(g, len(counts), N, K), offsets, rows


def check(x, w, offsets, rows, y):
    xs, ws, bounds = values64(x), values64(w), offsets.tolist()
    C = xs.shape[1]
    for e in range(ws.shape[0]):
        a, b = bounds[e], bounds[e + 1]
        xe = xs[rows[a:b].long()] if rows is not None else xs[a:b]
        size = xe.abs() @ ws[e].abs().T
        far = (y[a:b].double() - xe @ ws[e].T).abs() - size * (C * 2.0**-22 + UNIT[y.dtype]) - 2.0**-24
        assert torch.isfinite(y[a:b]).all() and (far <= 0).all(), (e, far.max().item())
    assert not y[bounds[-1]:].any()


COUNTS = {
    "one row": [1],
    "one each": [1] * 8,
    "empty groups": [0, 3, 0, 0, 17, 1, 0],
    "few, ragged": [5, 64, 0, 65, 2, 33, 16, 15],
    "even": [128, 128],
    "wide": [300, 0, 17, 600, 224, 1, 129, 225],
    "dense": [777],
    "none": [0, 0, 0],
}


@pytest.mark.parametrize("name", COUNTS)
@pytest.mark.parametrize("N,K", [(128, 256), (264, 32), (1416, 544), (7, 96), (384, 2048)])
def test_products(name, N, K):
    counts = COUNTS[name]
    x, w, offsets, rows = make(counts, N, K, seed=N + len(counts), tail=3)
    rows[sum(counts):] = -1
    y = expert_linear_mxfp4(x, w, offsets, rows=rows, dtype=torch.float32)
    check(x, w, offsets, rows, y)
    inside = rows.clamp(min=0).long()
    ordered = MxTensor(x.codes[inside].contiguous(), x.scales[inside].contiguous())
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        y2 = expert_linear_mxfp4(ordered, w, offsets, dtype=dtype)
        assert torch.equal(y2, y.to(dtype))  # the same sums, rounded to the type
    assert _native.device_wait_timeouts(reset=True) == 0


@pytest.mark.parametrize("counts,N,K", [([1], 256, 8192), ([3, 2], 64, 4128), ([16, 1, 0, 7], 136, 14336), ([64], 2048, 2304)])
def test_contractions_split_over_a_cluster(counts, N, K):
    x, w, offsets, rows = make(counts, N, K, seed=K)
    y = expert_linear_mxfp4(x, w, offsets, rows=rows)
    check(x, w, offsets, rows, y)
    assert torch.equal(expert_linear_mxfp4(x, w, offsets, rows=rows), y)
    assert _native.device_wait_timeouts(reset=True) == 0


# Rows on average where the tiles change (16 a group), with groups of more than a tile's rows.
@pytest.mark.parametrize("counts", [[16] * 4, [17, 16, 16, 16], [1, 60, 0, 3], [1, 60, 2, 3], [31, 33, 0, 0]])
@pytest.mark.parametrize("N,K", [(136, 800), (520, 2272)])
def test_sizes_where_the_tiles_change(counts, N, K):
    x, w, offsets, rows = make(counts, N, K, seed=sum(counts) + K)
    y = expert_linear_mxfp4(x, w, offsets, rows=rows, dtype=torch.float32)
    check(x, w, offsets, rows, y)
    ordered = MxTensor(x.codes[rows.long()].contiguous(), x.scales[rows.long()].contiguous())
    assert torch.equal(expert_linear_mxfp4(ordered, w, offsets, dtype=torch.float32), y)
    assert _native.device_wait_timeouts(reset=True) == 0


@pytest.mark.parametrize("counts", [[300, 0, 2, 209], [100, 417, 40]])
@pytest.mark.parametrize("K", [64, 2048, 2080])
def test_contractions_where_the_stores_change(counts, K):
    x, w, offsets, rows = make(counts, 520, K, seed=K, tail=2)
    rows[sum(counts):] = -1
    for dtype in (torch.float32, torch.bfloat16):
        check(x, w, offsets, rows, expert_linear_mxfp4(x, w, offsets, rows=rows, dtype=dtype))
    assert _native.device_wait_timeouts(reset=True) == 0


def test_large_products():
    x, w, offsets, rows = make([1500, 260, 2000, 3], 2048, 1024, seed=1)
    check(x, w, offsets, rows, expert_linear_mxfp4(x, w, offsets, rows=rows))


@pytest.mark.parametrize("counts", [[3, 2, 4], [300, 70, 200]])
def test_a_group_does_not_see_its_neighbours(counts):
    x, w, offsets, rows = make(counts, 200, 160, seed=7)
    y = expert_linear_mxfp4(x, w, offsets, rows=rows)
    lo, hi = offsets[1], offsets[2]
    w.scales[1] = 255
    y2 = expert_linear_mxfp4(x, w, offsets, rows=rows)
    assert torch.equal(y[:lo], y2[:lo]) and torch.equal(y[hi:], y2[hi:]) and torch.isnan(y2[lo:hi]).all()
    x.scales[3, 2] = 255  # one NaN block of one token
    y3 = expert_linear_mxfp4(x, w, offsets, rows=rows)
    hit = torch.isnan(y3).all(1)
    assert torch.equal(hit, (rows == 3) | ((torch.arange(len(rows), device="cuda") >= lo) & (torch.arange(len(rows), device="cuda") < hi)))
    assert torch.equal(y3[~hit], y[~hit])


@pytest.mark.parametrize("rows_at_most", [40, 900])
def test_wide_scales_and_zero_blocks(rows_at_most):
    # The scales' whole range, and blocks of zeros with the smallest one.
    g = torch.Generator(device="cuda").manual_seed(5)
    x, w = random_mx(g, rows_at_most, 256, low=-60, high=40), random_mx(g, 1, 96, 256, low=-40, high=20)
    x.codes[::3, 16:48], x.scales[::3, 1:3] = 0, 0
    offsets = torch.tensor([0, rows_at_most], dtype=torch.int32, device="cuda")
    check(x, w, offsets, None, expert_linear_mxfp4(x, w, offsets, dtype=torch.float32))


def test_layer_of_experts():
    # Quantised activations through two products, against the same steps on dequantised values.
    g = torch.Generator(device="cuda").manual_seed(11)
    T, E, k, H, I = 70, 6, 2, 128, 256
    h = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    up = mxfp4_quantize(torch.randn(E, I, H, generator=g, device="cuda") / math.sqrt(H))
    down = mxfp4_quantize(torch.randn(E, H, I, generator=g, device="cuda") / math.sqrt(I))
    r = route_experts(torch.randn(T, E, generator=g, device="cuda"), k)
    mid = torch.relu(expert_linear_mxfp4(mxfp4_quantize(h), up, r.offsets, rows=r.rows))
    mid4 = mxfp4_quantize(mid)
    out = combine_experts(expert_linear_mxfp4(mid4, down, r.offsets), r.weights, r.positions).double()
    values, want = mxfp4_dequantize(mid4, torch.float32).double(), torch.zeros(T, H, dtype=torch.float64, device="cuda")
    matrix = mxfp4_dequantize(down, torch.float32).double()
    for j in range(k):
        part = torch.einsum("ti,thi->th", values[r.positions[:, j].long()], matrix[r.experts[:, j].long()])
        want += r.weights[:, j, None].double() * part
    assert (out - want).norm() <= 2.0**-7 * want.norm()  # two roundings to BF16


def test_output_rows_of_a_wider_buffer():
    x, w, offsets, rows = make([20, 0, 30], 96, 128, seed=4)
    buffer = torch.full((50, 101), 7.0, device="cuda").bfloat16()
    out = expert_linear_mxfp4(x, w, offsets, rows=rows, out=buffer[:, 2:98])
    check(x, w, offsets, rows, out)
    assert (buffer[:, :2] == 7).all() and (buffer[:, 98:] == 7).all()
    wide = torch.full((50, 104), 7.0, device="cuda").half()
    check(x, w, offsets, rows, expert_linear_mxfp4(x, w, offsets, rows=rows, out=wide[:, :96]))
    assert (wide[:, 96:] == 7).all()


@pytest.mark.parametrize("tokens", [600, 20000])
def test_a_thousand_experts(tokens):
    g = torch.Generator(device="cuda").manual_seed(12)
    r = route_experts(torch.randn(tokens, 1024, generator=g, device="cuda"), 5)
    x, w = random_mx(g, tokens, 96), random_mx(g, 1024, 40, 96)
    check(x, w, r.offsets, r.rows, expert_linear_mxfp4(x, w, r.offsets, rows=r.rows))


def test_offsets_past_32_bits():
    # 2.4e9 codes' bytes, then 2.2e9 outputs: the last expert's rows against 64 bits.
    g = torch.Generator(device="cuda").manual_seed(14)
    E, N, K = 3, 32768, 49152
    w = random_mx(g, E, N, K)
    offsets = torch.tensor([0, 2, 3, 5], dtype=torch.int32, device="cuda")
    x = random_mx(g, 5, K)
    y = expert_linear_mxfp4(x, w, offsets, dtype=torch.float32)
    last = MxTensor(w.codes[2, -256:].contiguous(), w.scales[2, -256:].contiguous())
    xs, ws = values64(x)[3:], values64(last)
    assert ((y[3:, -256:].double() - xs @ ws.T).abs() <= (xs.abs() @ ws.abs().T) * K * 2.0**-22).all()
    del w, y
    R, N, K = 70000, 32000, 32
    x, w = random_mx(g, R, K), random_mx(g, 2, N, K)
    offsets = torch.tensor([0, 30000, R], dtype=torch.int32, device="cuda")
    y = expert_linear_mxfp4(x, w, offsets)
    xs, ws = values64(MxTensor(x.codes[-64:], x.scales[-64:])), values64(w)[1]
    far = (y[-64:].double() - xs @ ws.T).abs() - (xs.abs() @ ws.abs().T) * (K * 2.0**-22 + 2.0**-8)
    assert (far <= 2.0**-24).all()


@pytest.mark.parametrize("counts", [[3, 0, 2], [40, 300, 90]])
def test_other_streams_and_captured_graphs(counts):
    x, w, offsets, rows = make(counts, 136, 192, seed=13)
    want = expert_linear_mxfp4(x, w, offsets, rows=rows)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = expert_linear_mxfp4(x, w, offsets, rows=rows)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = expert_linear_mxfp4(x, w, offsets, rows=rows)
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)


def test_refusals():
    x, w, offsets, rows = make([4, 4], 64, 64, seed=2)
    with pytest.raises(TypeError, match="MxTensor"):
        expert_linear_mxfp4(tuple(x), w, offsets, rows=rows)
    with pytest.raises(ValueError, match="width"):
        expert_linear_mxfp4(MxTensor(x.codes[:, :16].contiguous(), x.scales[:, :1].contiguous()), w, offsets, rows=rows)
    with pytest.raises(ValueError, match="scales"):
        expert_linear_mxfp4(x, MxTensor(w.codes, w.scales[:, :32]), offsets, rows=rows)
    with pytest.raises(ValueError, match="offsets"):
        expert_linear_mxfp4(x, w, offsets[:-1], rows=rows)
    with pytest.raises(ValueError, match="dtype"):
        expert_linear_mxfp4(x, w, offsets, rows=rows, dtype=torch.float64)
    with pytest.raises(ValueError, match="out must"):
        expert_linear_mxfp4(x, w, offsets, rows=rows, out=torch.empty(7, 64, device="cuda").bfloat16())
    with pytest.raises(RuntimeError, match="workspace"):
        _native.call("lf_expert_linear_mxfp4", 2, 16, 16, 4, 16, 16, 16, 16, 1, 100, 64, 64, 16, 64, None, 0, None)


# A rank's part of the experts: rows before the first bound and from the last one on are of no group.
@pytest.mark.parametrize("counts,lo,hi", [([3, 0, 5, 2, 1, 4], 2, 5), ([9, 14, 17, 12, 11], 1, 3), ([40, 300, 90, 0, 260, 7], 1, 5),
                                          ([30, 70, 0, 0], 2, 4), ([600, 5], 1, 2)])
@pytest.mark.parametrize("by_index", [True, False])
@pytest.mark.parametrize("N,K,dtype", [(136, 192, torch.float32), (264, 1024, torch.bfloat16)])
def test_a_slice_of_the_experts(counts, lo, hi, by_index, N, K, dtype):
    x, w, offsets, rows = make(counts, N, K, seed=sum(counts) + lo, tail=2)
    rows[sum(counts):] = -1
    if not by_index:
        inside = rows.clamp(min=0).long()
        x, rows = MxTensor(x.codes[inside].contiguous(), x.scales[inside].contiguous()), None
    mine, part = MxTensor(w.codes[lo:hi], w.scales[lo:hi]), offsets[lo : hi + 1]
    y = torch.full((sum(counts) + 2, N), math.nan, device="cuda", dtype=dtype)
    expert_linear_mxfp4(x, mine, part, rows=rows, out=y)
    check(x, mine, part, rows, y)
    assert not y[: int(part[0])].any()
