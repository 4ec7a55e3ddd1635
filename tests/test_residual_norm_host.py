"""residual_norm's refusals: argument checks that need no GPU, in Python and at the C entry points."""

import ctypes

import pytest
import torch

from parallel_amd import _lib, residual_norm

BF = torch.bfloat16


@pytest.mark.parametrize("change,match", [
    (dict(residual=torch.zeros(4, 24, dtype=BF)), "does not match"),
    (dict(residual=torch.zeros(4, 16)), "residual must be"),
    (dict(weight=torch.zeros(8, dtype=BF)), "weight must be"),
    (dict(weight=torch.zeros(16)), "weight must be"),
    (dict(post_weight=torch.zeros(4, 16, dtype=BF)), "post_weight must be"),
    (dict(gate=torch.zeros(4, dtype=BF)), "gate must be"),
    (dict(gate=torch.zeros(1, 16, dtype=BF)), "gate must be"),
    (dict(gate=torch.zeros(4, 1)), "gate must be"),
    (dict(y=torch.zeros(4, 16, dtype=torch.float16), residual=torch.zeros(4, 16, dtype=torch.float16)), "float16"),
    ({}, "GPU only"),
])
def test_python_refusals(change, match):
    args = dict(y=torch.zeros(4, 16, dtype=BF), residual=torch.zeros(4, 16, dtype=BF), weight=torch.zeros(16, dtype=BF))
    with pytest.raises(ValueError, match=match):
        residual_norm(**{**args, **change})


def test_c_entry_points_check_their_arguments():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(256)
    b = ctypes.addressof(buf) + (16 - ctypes.addressof(buf) % 16) % 16

    def fwd(y=b, post=None, gate=None, kind=0, gamma=b, T=1, H=16, eps=1e-6, x=b, rstd_y=None):
        return lib.moe_residual_norm_fwd(y, b, post, gate, kind, gamma, 0, T, H, 1.0, 1.0, eps, b, x, rstd_y, b, None)

    assert fwd(T=0, y=None, x=None) == _lib.MOE_OK  # nothing to do, and no HIP call
    for bad in (dict(y=None), dict(gamma=None), dict(kind=4), dict(kind=1), dict(T=-1), dict(T=1 << 31), dict(eps=-1.0),
                dict(x=None), dict(y=b + 2), dict(x=b + 8), dict(post=b + 8), dict(gamma=b + 4)):
        assert fwd(**bad) == _lib.MOE_ERR_INVALID, bad
    for bad in (dict(H=12), dict(H=0), dict(H=8200)):
        assert fwd(**bad) == _lib.MOE_ERR_UNSUPPORTED, bad

    need = lib.moe_residual_norm_bwd_workspace_bytes(5000, 2048)
    assert need == 3 * 1024 * 2048 * 4
    assert lib.moe_residual_norm_bwd_workspace_bytes(5000, 512) == 3 * 4096 * 512 * 4
    assert lib.moe_residual_norm_bwd_workspace_bytes(0, 512) == 3 * 512 * 4

    def bwd(post=None, gate=None, kind=0, d_y=None, d_res=b, d_post=None, d_gate=None, d_gamma=b, ws=b, nbytes=192):
        return lib.moe_residual_norm_bwd(b, b, b, b, post, gate, kind, b, b, b, 0, 1, 16, 1.0, 1.0, d_y, d_res, d_post,
                                         d_gate, d_gamma, ws, nbytes, None)

    assert bwd(nbytes=191) == _lib.MOE_ERR_WORKSPACE and bwd(ws=None) == _lib.MOE_ERR_WORKSPACE
    for bad in (dict(d_gamma=None), dict(post=b, d_y=b), dict(gate=b, kind=2, d_y=b), dict(gate=b, kind=1, d_y=b),
                dict(gate=b, kind=1, d_gate=b), dict(d_res=None), dict(d_res=b + 2)):
        assert bwd(**bad) == _lib.MOE_ERR_INVALID, bad
