"""Refusals of the 4-bit operators, in Python and at the C entry points, and the oracle's own format: no GPU."""

import ctypes

import pytest
import torch

import mx4_oracle as O
from parallel_amd import MX4Experts, MX4Tensor, _lib, mx4_experts, mx4_grouped_mm, mx4_swiglu, quantize_mx4

U8 = torch.uint8


def mx(*shape):
    return MX4Tensor(torch.zeros(*shape[:-1], shape[-1] // 2, dtype=U8),
                     torch.zeros(*shape[:-1], 8 * -(-shape[-1] // 256), dtype=U8))


def test_tensor_checks_its_parts():
    t = mx(3, 96)
    assert t.shape == (3, 96) and t.block_scales.shape == (3, 3)
    assert MX4Tensor(t.codes, torch.zeros(3, 3, dtype=U8)).scales.shape == (3, 8)
    with pytest.raises(ValueError, match="whole blocks"):
        MX4Tensor(torch.zeros(3, 24, dtype=U8), torch.zeros(3, 8, dtype=U8))
    with pytest.raises(ValueError, match="do not match"):
        MX4Tensor(torch.zeros(3, 48, dtype=U8), torch.zeros(3, 16, dtype=U8))
    with pytest.raises(ValueError, match="do not match"):
        MX4Tensor(torch.zeros(3, 48, dtype=U8), torch.zeros(4, 8, dtype=U8))
    with pytest.raises(ValueError, match="uint8"):
        MX4Tensor(torch.zeros(3, 48, dtype=torch.int8), torch.zeros(3, 8, dtype=U8))
    with pytest.raises(ValueError, match="float16"):
        t.dequantize(torch.float16)


@pytest.mark.parametrize("call,match", [
    (lambda: quantize_mx4(torch.zeros(2, 40)), "whole blocks"),
    (lambda: quantize_mx4(torch.zeros(2, 32, dtype=torch.float16)), "float16"),
    (lambda: quantize_mx4(torch.zeros(2, 0)), "whole blocks"),
    (lambda: quantize_mx4(torch.zeros(2, 32)), "GPU only"),
    (lambda: mx(2, 64).dequantize(), "GPU only"),
    (lambda: mx4_grouped_mm(mx(4, 64), mx(2, 16, 96), torch.zeros(2, dtype=torch.int32)), "values a row"),
    (lambda: mx4_grouped_mm(mx(4, 64), mx(16, 64), torch.zeros(2, dtype=torch.int32)), "groups, N, K"),
    (lambda: mx4_grouped_mm(mx(4, 64), mx(2, 16, 64), torch.zeros(3, dtype=torch.int32)), "offsets"),
    (lambda: mx4_grouped_mm(mx(4, 64), mx(2, 16, 64), torch.zeros(2, dtype=torch.int64)), "offsets"),
    (lambda: mx4_swiglu(mx(4, 64), mx(2, 16, 64), torch.zeros(2, dtype=torch.int32)), "GPU only"),
    (lambda: mx4_experts(torch.zeros(4, 64), torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 3), mx(2, 64, 64),
                         mx(2, 64, 32)), "tokens, k"),
    (lambda: mx4_experts(torch.zeros(4, 64), torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2), mx(2, 64, 64),
                         mx(2, 64, 64)), "do not match"),
    (lambda: mx4_experts(torch.zeros(4, 64), torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2), mx(2, 64, 64),
                         mx(2, 64, 32)), "GPU only"),
    (lambda: MX4Experts(mx(2, 64, 64), mx(3, 64, 32)), "do not match"),
])
def test_python_refusals(call, match):
    with pytest.raises(ValueError, match=match):
        call()


def test_c_entry_points_check_their_arguments():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(256)
    b = ctypes.addressof(buf) + (16 - ctypes.addressof(buf) % 16) % 16
    OK, INV, UNS = _lib.MOE_OK, _lib.MOE_ERR_INVALID, _lib.MOE_ERR_UNSUPPORTED

    for name, fn in (("q", lambda x=b, r=1, k=32, c=b, s=b: lib.moe_mx4_quantize(x, 0, r, k, c, s, None)),
                     ("d", lambda x=b, r=1, k=32, c=b, s=b: lib.moe_mx4_dequantize(c, s, r, k, 0, x, None))):
        assert fn(x=None, c=None, s=None, r=0) == OK, name
        for bad in (dict(x=None), dict(c=None), dict(s=None), dict(r=-1), dict(k=0), dict(x=b + 8), dict(c=b + 4),
                    dict(s=b + 4)):
            assert fn(**bad) == INV, (name, bad)
        for bad in (dict(k=48), dict(r=1 << 40, k=64)):
            assert fn(**bad) == UNS, (name, bad)

    def mm(a=b, sa=b, rows=4, idx=None, div=1, w=b, sw=b, offs=b, G=2, M=4, N=16, K=64, c=b):
        return lib.moe_mx4_grouped_gemm(a, sa, rows, idx, div, w, sw, offs, G, M, N, K, c, None)

    assert mm(M=0, rows=0, a=None, sa=None, c=None) == OK
    for bad in (dict(a=None), dict(sa=None), dict(w=None), dict(sw=None), dict(offs=None), dict(c=None), dict(G=0),
                dict(M=-1), dict(N=0), dict(K=0), dict(div=0), dict(rows=3), dict(rows=-1), dict(a=b + 8),
                dict(sa=b + 4), dict(w=b + 8), dict(sw=b + 2), dict(c=b + 8)):
        assert mm(**bad) == INV, bad
    for bad in (dict(K=48), dict(N=12), dict(M=1 << 31, rows=1 << 31), dict(K=1 << 28, rows=64, M=64),
                dict(N=1 << 20, K=1 << 12), dict(G=1 << 24)):
        assert mm(**bad) == UNS, bad

    def glu(I=32, act=None, codes=b, scales=b, M=4):
        return lib.moe_mx4_grouped_swiglu(b, b, 4, None, 1, b, b, b, 2, M, I, 64, act, codes, scales, None)

    assert glu(M=0) == OK
    assert glu(I=40) == UNS  # not whole blocks of 32 in 4 bits
    assert glu(scales=None) == INV and glu(codes=b + 8) == INV and glu(codes=None) == INV


def test_experts_entry_point_checks_its_arguments():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(256)
    b = ctypes.addressof(buf) + (16 - ctypes.addressof(buf) % 16) % 16
    OK, INV, UNS = _lib.MOE_OK, _lib.MOE_ERR_INVALID, _lib.MOE_ERR_UNSUPPORTED

    def experts(x=b, f32=0, ids=b, w=b, T=4, H=64, k=2, E=4, I=32, guc=b, gus=b, dnc=b, dns=b, out=b, ws=b, size=1 << 40):
        return lib.moe_mx4_experts(x, f32, ids, w, T, H, k, E, I, guc, gus, dnc, dns, out, ws, size, None)

    def size(f32=0, T=4, H=64, k=2, E=4, I=32):
        return lib.moe_mx4_experts_workspace_bytes(f32, T, H, k, E, I)

    assert experts(T=0, x=None, ids=None, w=None, guc=None, gus=None, dnc=None, dns=None, out=None, ws=None, size=0) == OK
    pointers = (dict(x=None), dict(ids=None), dict(w=None), dict(out=None), dict(x=b + 8), dict(out=b + 8),
                dict(guc=None), dict(gus=None), dict(dnc=None), dict(dns=None), dict(guc=b + 8), dict(gus=b + 4),
                dict(dnc=b + 8), dict(dns=b + 4))
    for bad in (dict(T=-1), dict(H=0), dict(I=0), dict(k=0), dict(k=17), dict(E=0), dict(H=1 << 21), dict(I=1 << 21),
                dict(T=1 << 31), dict(T=1 << 28, k=8)) + pointers + tuple(dict(T=100, **p) for p in pointers):
        assert experts(**bad) == INV, bad
        if not any(name in bad for name in ("x", "ids", "w", "out", "guc", "gus", "dnc", "dns")):
            assert size(**bad) == 0, bad
    # rows that are not whole blocks, more experts than the sort takes (also where nothing is sorted), 2 GiB
    for bad in (dict(H=48), dict(I=40), dict(E=1025), dict(E=1025, T=1), dict(H=1 << 16, I=1 << 15, T=1),
                dict(T=1 << 26, H=64, k=1), dict(T=1 << 24, I=1 << 9, k=8)):
        assert experts(**bad) == UNS, bad
    for T in (4, 100):  # without and with the sort
        for f32 in (0, 1):
            need = size(f32, T)
            assert need > 0
            assert experts(T=T, f32=f32, size=need - 1) == _lib.MOE_ERR_WORKSPACE
            assert experts(T=T, f32=f32, ws=None) == _lib.MOE_ERR_WORKSPACE
            assert experts(T=T, f32=f32, ws=b + 8) == _lib.MOE_ERR_WORKSPACE


def test_oracle_follows_the_format():
    """Blocks written out by hand: scale rule, ties, saturation, sign, NaN, packing order."""
    x = torch.zeros(3, 32)
    x[0, :9] = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -7.9])  # largest 7.9: e = 0
    x[1, 0] = 2.0 ** -130
    x[2, 3] = float("inf")
    idx, s = O.quantize(x)
    assert s[:, 0].tolist() == [127, 0, 255]
    assert idx[0, :9].tolist() == [6, 0, 2, 2, 4, 4, 6, 6, 15]
    assert idx[1, 0].item() == 0 and not idx[2].any()  # 2^-130 / 2^-127 = 1/8 rounds to 0
    assert O.pack(idx)[0, 0].item() == 6 and O.pack(idx)[0, 1].item() == (2 | 2 << 4)
    assert torch.equal(O.unpack(O.pack(idx)), idx)
    assert O.values(idx, s)[0, :2].tolist() == [4.0, 0.0] and O.values(idx, s)[0, 8].item() == -6.0
    assert torch.isnan(O.values(idx, s)[2]).all()
