"""What the cache of 8 bits refuses, on the CPU: nothing of it reaches a kernel."""
import pytest
import torch

from vosti_b200 import ops


def parts(pages=2, heads=2, page=32, d=64, device="cpu"):
    return list(ops.PagedE4M3.tensors(pages, heads, page, d, torch.device(device)))


def test_empty_cache():
    k, v, k_scale, v_scale = parts()
    assert tuple(k.shape) == (2, 2, 32, 64) and tuple(v.shape) == (2, 2, 2, 64, 16) and tuple(k_scale.shape) == tuple(v_scale.shape) == (2, 2, 2)
    assert k.dtype == v.dtype == torch.float8_e4m3fn and k_scale.dtype == v_scale.dtype == torch.float8_e8m0fnu
    for page in (0, 8, 24, -16):
        with pytest.raises(ops.KernelError):
            ops.PagedE4M3.tensors(2, 2, page, 64, torch.device("cpu"))


def test_cache_shapes_and_types():
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.PagedE4M3(*parts())
    good = parts()
    for i, bad in ((0, good[0][0]), (0, good[0][..., :40].contiguous()), (0, good[0][:, :, :24].contiguous()), (1, good[0]), (2, good[2][:1]), (3, good[3][:, :, :1]),
                   (0, good[0].view(torch.uint8)), (1, good[1].float()), (2, good[2].view(torch.uint8)), (3, good[3].float())):
        with pytest.raises(ops.KernelError):
            ops.PagedE4M3(*(bad if i == at else t for at, t in enumerate(good)))


def test_plain_numbers():
    """The test's own reading of the formats against torch's."""
    import plain_e4m3 as plain
    b = torch.arange(256, dtype=torch.uint8)
    a, c = plain.held(b.view(torch.float8_e4m3fn)), b.view(torch.float8_e4m3fn).double()
    assert torch.equal(a.nan_to_num(7e9), c.nan_to_num(7e9))
    a, c = plain.scales(b.view(torch.float8_e8m0fnu)), b.view(torch.float8_e8m0fnu).float().double()
    assert torch.equal(a.nan_to_num(0.5), c.nan_to_num(0.5))
    for most in (1e-40, 3e-39, 1e-30, 447.9, 448.0, 448.1, 3e38):
        s = 2.0 ** (plain.scale_for(most) - 127)
        assert most / s <= 448 and (most / s > 224 or plain.scale_for(most) == 0)
