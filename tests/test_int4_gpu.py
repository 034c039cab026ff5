"""Products with 4-bit weights on the GPU against 64 bits.

Bounds. Up to 16 rows a group's codes meet the rows exactly, sums are float32: off by (k + group count) 2^-24 of sum |x||w| at most. With more
rows codes times scales are rounded to bfloat16, 2^-8 of each product at most; then the same sums. The result's rounding is 2^-8 of it in
bfloat16, 2^-24 in float32."""
import pytest
import torch

from vosti_b200 import ops

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"


def weight(features, k, group, seed=0):
    gen = torch.Generator().manual_seed(seed + features + k)
    codes = torch.randint(-8, 8, (features, k), generator=gen, dtype=torch.int8)
    scales = (torch.rand(features, -(-k // group), generator=gen) * 0.01 + 0.001).bfloat16()
    return ops.Int4Weight.from_codes(codes.to(DEVICE), scales.to(DEVICE), group), codes.double() * scales.double().repeat_interleave(group, dim=1)[:, :k], gen


def check(y, x, w, rows):
    want, size = x.double() @ w.T, x.double().abs() @ w.abs().T
    bound = (x.shape[1] + 8) * 2.0 ** -24 * size + (2.0 ** -8 if y.dtype == torch.bfloat16 else 2.0 ** -24) * want.abs()
    if rows > 16:
        bound += 2.0 ** -8 * size
    worst = float(((y.cpu().double() - want).abs() - bound).max())
    assert worst <= 0, worst


@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 16, 17, 33, 64, 65, 128, 129, 256, 300])
@pytest.mark.parametrize("features,k,group", [(16, 128, 128), (1000, 1024, 128), (130, 640, 32), (4096, 512, 64), (33, 4096, 128), (257, 96, 32), (5000, 2048, 64),
                                              (1, 64, 64), (640, 200, 32)])
def test_products(rows, features, k, group):
    w, numbers, gen = weight(features, k, group)
    x = torch.randn(rows, k, generator=gen).bfloat16()
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    for kind in (torch.bfloat16, torch.float32):
        y = ops.gemm_int4(x.to(DEVICE), w, status, out_dtype=kind)
        assert int(status) == 0 and y.dtype == kind and tuple(y.shape) == (rows, features)
        check(y, x, numbers, rows)


@pytest.mark.parametrize("rows", [1, 16, 17, 40])
@pytest.mark.parametrize("k", [1, 7, 100, 129, 1003])
def test_rows_that_start_inside_a_word(rows, k):
    w, numbers, gen = weight(70, k, 32)
    x = torch.randn(rows, k, generator=gen).bfloat16()
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    check(ops.gemm_int4(x.to(DEVICE), w, status), x, numbers, 17)
    # the same matrix from an odd address
    odd = torch.zeros(rows * 128 + 1, dtype=torch.bfloat16, device=DEVICE)[1:].view(rows, 128)
    w, numbers, gen = weight(70, 128, 32)
    x = torch.randn(rows, 128, generator=gen).bfloat16()
    odd.copy_(x)
    check(ops.gemm_int4(odd, w, status), x, numbers, 17)


def test_no_rows():
    w, _, _ = weight(32, 128, 128)
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    assert tuple(ops.gemm_int4(torch.empty(0, 128, dtype=torch.bfloat16, device=DEVICE), w, status).shape) == (0, 32)


@pytest.mark.parametrize("rows", [3, 60])
def test_what_stands_beyond_the_matrix_does_not_count(rows):
    w, numbers, gen = weight(40, 200, 32)
    w.codes.view(3, 2, 16, 4, 4, 4)[2, :, 8:] = 255                       # rows 40 .. 47
    w.scales[2, :, 8:] = float("nan")
    w.scales[:, 1, :, 3] = float("nan")                                   # k 224 .. 255
    x = torch.randn(rows, 200, generator=gen).bfloat16()
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    check(ops.gemm_int4(x.to(DEVICE), w, status), x, numbers, rows)


@pytest.mark.parametrize("rows", [2, 20])
def test_rows_do_not_mix(rows):
    """A row that is no number leaves the others alone."""
    w, numbers, gen = weight(200, 512, 128)
    x = torch.randn(rows, 512, generator=gen).bfloat16()
    x[1, 7] = float("nan")
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    y = ops.gemm_int4(x.to(DEVICE), w, status).cpu()
    assert y[1].isnan().all()
    keep = [r for r in range(rows) if r != 1]
    check(y[keep], x[keep], numbers, rows)


def test_another_stream_and_a_graph():
    w, _, gen = weight(512, 1024, 128)
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    for rows in (4, 70):
        x = torch.randn(rows, 1024, generator=gen).bfloat16().to(DEVICE)
        want = ops.gemm_int4(x, w, status)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = ops.gemm_int4(x, w, status)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = ops.gemm_int4(x, w, status)
        kept.zero_()
        graph.replay()
        assert torch.equal(kept, want)


def test_quantized_on_the_device():
    gen = torch.Generator().manual_seed(5)
    w = torch.randn(130, 300, generator=gen) * 0.02
    a, b = ops.Int4Weight.quantize(w, 64), ops.Int4Weight.quantize(w.to(DEVICE), 64)
    assert torch.equal(a.codes, b.codes.cpu()) and torch.equal(a.scales, b.scales.cpu())


def test_tiles_ask_for_no_more_tensor_memory_than_an_sm_has():
    for tile in range(4):
        assert 0 < ops.library().vosti_gemm_int4_columns_an_sm(tile) <= 512
    assert ops.library().vosti_gemm_int4_columns_an_sm(4) == -1


def test_calls_that_are_refused():
    w, _, gen = weight(64, 256, 64)
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    x = torch.randn(5, 256, generator=gen).bfloat16().to(DEVICE)
    ops.gemm_int4(x, w, status)
    for bad in (x[0], x.float(), x.cpu(), x[:, :128].contiguous(), x[:, ::2], x.t().contiguous().t()):
        with pytest.raises(ops.KernelError):
            ops.gemm_int4(bad, w, status)
    for more in (dict(out_dtype=torch.float16), dict(out_dtype=torch.uint8)):
        with pytest.raises(ops.KernelError):
            ops.gemm_int4(x, w, status, **more)
    for bad in (status.cpu(), status.float(), status[:0]):
        with pytest.raises(ops.KernelError):
            ops.gemm_int4(x, w, bad)
    assert int(status) == 0


@pytest.mark.parametrize("rows", [1, 8, 9, 16, 17, 64, 130, 300])
@pytest.mark.parametrize("inter,k,group", [(16, 128, 128), (48, 200, 32), (1040, 512, 64), (12288, 1024, 128), (320, 4096, 32)])
def test_gated_products(rows, inter, k, group):
    """silu(gate) * up of blocks of 16 rows each. silu(g) moves by 1.1 times what g is off by at most, exp by (2 + 1.16 |g|) 2^-23 of itself and the
    division and products by 2^-23."""
    w, numbers, gen = weight(2 * inter, k, group)
    x = torch.randn(rows, k, generator=gen).bfloat16()
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    sums = x.double() @ numbers.T
    off = (k + 8) * 2.0 ** -24 * (x.double().abs() @ numbers.abs().T) + (2.0 ** -8 * (x.double().abs() @ numbers.abs().T) if rows > 16 else 0)
    (g, u), (dg, du) = (m.view(rows, inter // 16, 2, 16).permute(2, 0, 1, 3).reshape(2, rows, inter) for m in (sums, off))
    want = g * torch.sigmoid(g) * u
    for kind in (torch.bfloat16, torch.float32):
        y = ops.gemm_int4(x.to(DEVICE), w, status, out_dtype=kind, swiglu=True)
        assert int(status) == 0 and y.dtype == kind and tuple(y.shape) == (rows, inter)
        exact = (5 + 1.16 * g.abs()) * 2.0 ** -23 * want.abs() + 1.1 * dg * (u.abs() + du) + (g * torch.sigmoid(g)).abs() * du
        bound = exact + (2.0 ** -8 if kind == torch.bfloat16 else 2.0 ** -24) * (want.abs() + exact) + 1e-37
        assert bool(((y.cpu().double() - want).abs() <= bound).all())


def test_gated_products_that_are_refused():
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    for features, k in ((48, 128), (64, 100)):
        w, _, _ = weight(features, k, 32)
        with pytest.raises(ops.KernelError):
            ops.gemm_int4(torch.zeros(3, k, dtype=torch.bfloat16, device=DEVICE), w, status, swiglu=True)
    w, _, _ = weight(64, 128, 32)
    odd = torch.zeros(3 * 128 + 1, dtype=torch.bfloat16, device=DEVICE)[1:].view(3, 128)
    with pytest.raises(ops.KernelError):
        ops.gemm_int4(odd, w, status, swiglu=True)
    assert tuple(ops.gemm_int4(odd[:0], w, status).shape) == (0, 64) and int(status) == 0


@pytest.mark.parametrize("features,k,group", [(16, 128, 128), (130, 640, 32), (257, 96, 32), (333, 264, 64), (4096, 512, 64), (20, 1024, 128)])
@pytest.mark.parametrize("rows", [5, 16, 17, 64, 128, 129, 300])
def test_each_weight_alone(features, k, group, rows):
    """Rows of a single one pick single weights: codes times scales to the bit, rounded once to bfloat16 above 16 rows and not at all below."""
    w, numbers, _ = weight(features, k, group)
    numbers = (numbers.float().bfloat16() if rows > 16 else numbers.float()).to(DEVICE)      # (a code of 4 bits times 8 bits is exact in float32)
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    for start in range(0, k, rows):
        at = torch.arange(start, start + rows, device=DEVICE) * 7 % k
        x = torch.zeros(rows, k, dtype=torch.bfloat16, device=DEVICE)
        x[torch.arange(rows, device=DEVICE), at] = 1
        assert torch.equal(ops.gemm_int4(x, w, status, out_dtype=torch.float32), numbers[:, at].T.float())
    assert int(status) == 0


@pytest.mark.parametrize("rows", [17, 33, 64, 65, 128, 129, 300])
@pytest.mark.parametrize("features,k,group", [(1000, 1024, 128), (130, 640, 32), (4096, 512, 64), (257, 96, 32), (640, 200, 32), (300, 8192, 128)])
def test_products_of_rounded_weights(rows, features, k, group):
    """More than 16 rows against the weights as they are rounded: what is left are the float32 sums, each addition of which may be cut off
    below its last bit (2^-23 of at most sum |x||w|), and the result's rounding."""
    w, numbers, gen = weight(features, k, group, seed=3)
    rounded = numbers.float().bfloat16().double()
    x = torch.randn(rows, k, generator=gen).bfloat16()
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    want, size = x.double() @ rounded.T, x.double().abs() @ rounded.abs().T
    for kind, half in ((torch.float32, 2.0 ** -24), (torch.bfloat16, 2.0 ** -8)):
        y = ops.gemm_int4(x.to(DEVICE), w, status, out_dtype=kind).cpu().double()
        sums = (k + 8) * 2.0 ** -23 * size
        assert bool(((y - want).abs() <= sums + half * (want.abs() + sums)).all()) and int(status) == 0


@pytest.mark.parametrize("rows", [1, 16, 17, 40])
@pytest.mark.parametrize("k", [1, 7, 100, 129, 1003])
def test_rows_that_start_inside_a_word_are_exact(rows, k):
    """They take the few rows' kernel sixteen at a time, whose codes and scales are not rounded."""
    w, numbers, gen = weight(70, k, 32)
    x = torch.randn(rows, k, generator=gen).bfloat16()
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    for kind in (torch.float32, torch.bfloat16):
        check(ops.gemm_int4(x.to(DEVICE), w, status, out_dtype=kind), x, numbers, 16)
    assert int(status) == 0
