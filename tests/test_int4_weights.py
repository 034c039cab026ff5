"""Weights in 4 bits on the CPU: packing, rounding and refusals."""
import pytest
import torch

from vosti_b200 import ops


@pytest.mark.parametrize("features,k,group", [(16, 128, 128), (33, 200, 32), (5, 64, 64), (40, 513, 128), (1, 1, 32)])
def test_packing(features, k, group):
    gen = torch.Generator().manual_seed(k)
    codes = torch.randint(-8, 8, (features, k), generator=gen, dtype=torch.int8)
    scales = torch.rand(features, -(-k // group), generator=gen).bfloat16()
    w = ops.Int4Weight.from_codes(codes, scales, group)
    assert w.shape == (features, k) and w.group == group
    assert torch.equal(w.dequantized(), codes.float() * scales.float().repeat_interleave(group, dim=1)[:, :k])
    # one code by the layout's description
    for f, c in ((0, 0), (features - 1, k - 1), (features // 2, k // 3)):
        i, j, offset = c % 128 // 32, c % 32 // 8, c % 8
        word = int.from_bytes(bytes(w.codes[f // 16, c // 128, f % 16, j, i].tolist()), "little")
        nibble = offset // 2 if offset % 2 == 0 else (offset + 7) // 2
        assert (word >> (4 * nibble)) % 16 - 8 == int(codes[f, c])


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rounding(group, dtype):
    """A code is the nearest: off by half a step; the scale's own rounding (2^-8) may cut the largest by 7 * 2^-8 of a step."""
    w = (torch.randn(50, 320, generator=torch.Generator().manual_seed(1)) * 0.02).to(dtype)
    w[3, :128] = 0
    q = ops.Int4Weight.quantize(w, group)
    step = torch.nn.functional.pad(w.float(), (0, -320 % group)).view(50, -1, group).abs().amax(-1) / 7
    step = step.repeat_interleave(group, dim=1)[:, :320]
    assert bool(((q.dequantized() - w.float()).abs() <= step * (0.5 + 2.0 ** -7)).all())
    assert bool((q.dequantized()[3, :128 // group * group] == 0).all())


def test_refusals():
    codes, scales = torch.zeros(16, 128, dtype=torch.int8), torch.ones(16, 1)
    for group in (0, 16, 256, -128):
        with pytest.raises(ops.KernelError, match="group"):
            ops.Int4Weight.from_codes(codes, scales, group)
        with pytest.raises(ops.KernelError, match="group"):
            ops.Int4Weight.quantize(scales, group)
    with pytest.raises(ops.KernelError):
        ops.Int4Weight.from_codes(codes.float(), scales, 128)
    with pytest.raises(ops.KernelError):
        ops.Int4Weight.from_codes(codes, scales, 64)
    with pytest.raises(ops.KernelError):
        ops.Int4Weight.quantize(torch.zeros(3), 128)
    with pytest.raises(ops.KernelError, match="finite"):
        ops.Int4Weight.quantize(torch.full((2, 128), float("inf")), 128)
    good = ops.Int4Weight.from_codes(codes, scales, 128)
    for bad in ((good.codes[..., :2], good.scales, good.shape), (good.codes.int(), good.scales, good.shape), (good.codes, good.scales.float(), good.shape),
                (good.codes, good.scales, (17, 128)), (good.codes, good.scales, (16, 129)), (good.codes, good.scales, (0, 128)),
                (good.codes, good.scales.expand(1, 1, 16, 3).contiguous(), good.shape)):
        with pytest.raises(ops.KernelError):
            ops.Int4Weight(*bad)


@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64])
def test_codes_of_other_quantizers(dtype):
    """Codes beyond -8 .. 7 would stand for others and reach into their neighbours' nibbles: refused, whatever their type."""
    scales = torch.ones(16, 1)
    for bad in (8, 15, 255, -9, -248, 2 ** 32):
        info = torch.iinfo(dtype)
        if info.min <= bad <= info.max:
            codes = torch.zeros(16, 128, dtype=dtype)
            codes[3, 77] = bad
            with pytest.raises(ops.KernelError, match="-8 .. 7"):
                ops.Int4Weight.from_codes(codes, scales, 128)
    codes = (torch.arange(16 * 128).view(16, 128) % 16).to(dtype) % 8
    assert torch.equal(ops.Int4Weight.from_codes(codes, scales, 128).dequantized(), codes.float())


def test_scales_and_types_that_are_refused():
    codes = torch.zeros(16, 128, dtype=torch.int8)
    for bad in (float("nan"), float("inf"), 3.4e38):               # (the last is infinite in bfloat16)
        scales = torch.ones(16, 1)
        scales[5] = bad
        with pytest.raises(ops.KernelError, match="finite"):
            ops.Int4Weight.from_codes(codes, scales, 128)
    for args in ((codes.bool(), torch.ones(16, 1)), (codes, torch.ones(16, 1, dtype=torch.int32)), (codes[:0], torch.ones(0, 1)), (codes[:, :0], torch.ones(16, 0)),
                 (codes.to(torch.complex64), torch.ones(16, 1))):
        with pytest.raises(ops.KernelError):
            ops.Int4Weight.from_codes(*args, 128)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("hidden,heads,kv,d,inter", [(256, 4, 2, 64, 512), (200, 5, 1, 48, 328)])
def test_bytes_that_the_benchmark_counts(group, hidden, heads, kv, d, inter):
    """The benchmark's closed form of a step's weight bytes against the weights' own tensors."""
    import bench
    config = dict(num_hidden_layers=3, hidden_size=hidden, num_attention_heads=heads, num_key_value_heads=kv, head_dim=d, intermediate_size=inter, vocab_size=300)
    matrices = [((heads + 2 * kv) * d, hidden), (hidden, heads * d), (2 * inter, hidden), (hidden, inter)]
    rest = 2 * (3 * (2 * hidden + 2 * d) + hidden + 300 * hidden)
    packed = [ops.Int4Weight.quantize(torch.ones(shape), group) for shape in matrices]
    assert bench.closed_form_weight_bytes(config, "int4", group) == rest + 3 * sum(w.codes.numel() + 2 * w.scales.numel() for w in packed)
    assert bench.closed_form_weight_bytes(config) == rest + 3 * sum(2 * f * k for f, k in matrices)
