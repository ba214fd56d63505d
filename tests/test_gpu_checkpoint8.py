"""pack8 / unpack8 on the native kernels: the codes are exact, so every comparison is for equality."""
import pytest
import torch

import gn_refs as R
from rdna4_conv3d import _native
from rdna4_conv3d.checkpoint8 import _pack_torch, pack8, unpack8
from test_group_norm_cpu import special

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_same_codes_as_on_the_cpu(cuda_ready, dtype, fmt):
    x = special(dtype)
    want = _pack_torch(x, fmt)
    n0 = _native.launch_count()
    p = pack8(x.cuda(), fmt)
    v = unpack8(p)
    assert _native.launch_count() - n0 == 2
    assert torch.equal(p.codes.cpu(), want[0]) and torch.equal(p.exponents.cpu(), want[1])
    limit = torch.finfo(dtype).max
    torch.testing.assert_close(v.cpu(), R.blocks64(x, fmt).clamp(-limit, limit).to(dtype), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("count", [1, 7, 8, 9, 31, 32, 33, 255, 1000, 8 * 32 * 37 + 5, 3000001])
def test_lengths(cuda_ready, count, dtype):
    g = torch.Generator(device="cuda").manual_seed(count)
    x = torch.randn(count, device="cuda", generator=g).to(dtype)
    for fmt in ("int8", "e4m3"):
        assert torch.equal(unpack8(pack8(x, fmt)), R.blocks64(x, fmt).to(dtype))


@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_every_code(cuda_ready, dtype):
    """All 256 codes under every exponent that a pack of this type can write."""
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").repeat(1, 1)
    for fmt in ("int8", "e4m3"):
        for byte in (0, 1, 90, 102, 103, 104, 127, 133, 134, 135, 136, 137, 200, 245, 246, 247, 248, 249):
            exps = torch.full((8,), byte, dtype=torch.uint8, device="cuda")
            from rdna4_conv3d.checkpoint8 import Packed8, _unpack_torch
            p = Packed8(codes.reshape(-1), exps, torch.Size((256,)), (1,), dtype, fmt)
            want = _unpack_torch(codes.reshape(-1).cpu(), exps.cpu(), fmt, torch.empty(256, dtype=dtype))
            torch.testing.assert_close(unpack8(p).cpu(), want, rtol=0, atol=0, equal_nan=True)


def test_layouts_and_alignment(cuda_ready):
    x = torch.randn(2, 5, 3, 4, 7, device="cuda").to(BF)
    wide = torch.zeros(x.numel() + 3, device="cuda", dtype=BF)
    off = wide[3:].copy_(x.reshape(-1)).reshape(x.shape)
    for t in (x, x.contiguous(memory_format=torch.channels_last_3d), x.permute(4, 2, 0, 1, 3), x[:, 1:3], x[..., ::2], off,
              x[0, 0, 0, 0, :1].expand(3, 6), x[0, 0, 0, 0, 0], x[:0]):
        p = pack8(t, "int8")
        v = unpack8(p)
        assert v.shape == t.shape and v.stride() == p.stride
        flat = v.as_strided((v.numel(),), (1,))
        mine = (t if p.stride == t.stride() else t.contiguous())
        assert torch.equal(flat, R.blocks64(mine.as_strided((t.numel(),), (1,)), "int8").to(BF))
    p = pack8(x)
    shifted = torch.zeros(p.codes.numel() + 1, dtype=torch.uint8, device="cuda")
    shifted[1:] = p.codes
    assert torch.equal(unpack8(p._replace(codes=shifted[1:])), unpack8(p))


def test_streams_and_graph(cuda_ready):
    x = torch.randn(1 << 20, device="cuda").to(HF)
    want = unpack8(pack8(x, "e4m3"))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = unpack8(pack8(x, "e4m3"))
    s.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = unpack8(pack8(x, "e4m3"))
    x.mul_(-2)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want * -2)


def test_past_32_bits(cuda_ready):
    count = (1 << 32) + 77
    x = torch.zeros(count, device="cuda", dtype=BF)
    tail = torch.randn(1001, device="cuda").to(BF)
    x[-1001:] = tail
    p = pack8(x)
    start = (count - 1001) // 32 * 32
    assert torch.equal(p.codes[start:], pack8(x[start:].clone()).codes)
    v = unpack8(p)
    assert torch.equal(v[-1001:], R.blocks64(x[start:], "int8").to(BF)[-1001:]) and not bool(v[:start].any())


def test_refusals_on_the_device(cuda_ready):
    x = torch.randn(40, device="cuda")
    p = pack8(x)
    for error, fn in ((TypeError, lambda: pack8(x.double())), (ValueError, lambda: pack8(x, "fp8")),
                      (ValueError, lambda: unpack8(p._replace(exponents=p.exponents.cpu()))),
                      (ValueError, lambda: unpack8(p._replace(codes=p.codes[1:])))):
        with pytest.raises(error):
            fn()
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            pack8(fwAD.make_dual(x, x))
