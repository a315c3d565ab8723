"""residual_norm refuses what it does not compute before anything is launched
(no GPU needed: the checks of shapes and types come before the device's)."""
import ctypes

import pytest
import torch

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def lib():
    from gpa_vggt_b200 import _lib, build
    build.build()
    return _lib.load()


def _t(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("error,args,kw", [
    (ValueError, (_t(2, 16), _t(2, 24)), {}),                                        # shapes differ
    (TypeError, (_t(2, 16), _t(2, 16, dtype=F32)), {}),                              # branch wider than the stream
    (TypeError, (_t(2, 16).half(), _t(2, 16).half()), {}),                           # fp16
    (ValueError, (_t(2, 12), _t(2, 12)), {}),                                        # columns not a multiple of 8
    (ValueError, (_t(1, 8200), _t(1, 8200)), {}),                                    # too wide
    (ValueError, (_t(2, 16), _t(2, 16)), dict(kind="batch")),
    (ValueError, (_t(2, 16), _t(2, 16)), dict(kind=None, weight=_t(16))),            # parameters without a norm
    (ValueError, (_t(2, 16), _t(2, 16)), dict(post_bias=_t(16))),
    (ValueError, (_t(2, 16), _t(2, 16)), dict(weight=_t(8))),
    (TypeError, (_t(2, 16), _t(2, 16)), dict(weight=_t(16), bias=_t(16, dtype=F32))),   # mixed parameter types
    (ValueError, (_t(2, 3, 16), _t(2, 3, 16)), dict(gate=_t(8))),
    (ValueError, (_t(2, 3, 16), _t(2, 3, 16)), dict(gate=_t(3, 16))),                # rank of neither form
    (ValueError, (_t(2, 3, 16), _t(2, 3, 16)), dict(gate=_t(1, 3, 16))),             # shared over leading dims
    (TypeError, (_t(2, 16), _t(2, 16)), dict(gate=_t(16).half())),
    (ValueError, (_t(2, 16), _t(2, 16)), dict(weight=_t(16))),                       # all well, but on the CPU
])
def test_refusals(error, args, kw):
    from gpa_vggt_b200 import kernels
    with pytest.raises(error, match="residual_norm"):
        kernels.residual_norm(*args, **kw)


def test_c_entry_refusals(lib):
    ok, odd = ctypes.c_void_p(256), ctypes.c_void_p(264)

    def fwd(x=ok, xd=1, xs=64, yd=1, ys=64, gate=None, gd=1, gate_rows=0, rows=4, cols=64, post=0, kind=1, pd=1,
            z=ok, h=ok, w=None):
        return lib.gpa_residual_norm(x, xd, xs, ok, yd, ys, gate, gd, gate_rows, rows, cols, post, None, None,
                                     1e-6, kind, w, None, pd, 1e-6, z, 64, h, 64, None, None)
    assert fwd(rows=0) == 0                       # nothing to do
    assert fwd(rows=-1) == 1 and fwd(cols=0) == 1
    assert fwd(cols=60) == 3 and fwd(cols=8200) == 3
    assert fwd(gate=ok, gate_rows=3) == 1         # does not divide the rows
    assert fwd(gate=ok, gate_rows=0) == 1
    assert fwd(xd=2) == 1 and fwd(yd=0) == 3      # unknown type; fp32 branch on a bf16 stream
    assert fwd(post=3) == 1 and fwd(kind=-1) == 1
    assert fwd(x=odd) == 1 and fwd(xs=60) == 1 and fwd(z=None) == 1 and fwd(h=None) == 1
    assert fwd(w=odd) == 1 and b"16-byte" in lib.gpa_last_error()

    size = lib.gpa_residual_norm_backward_workspace_bytes(4, 64, 4)
    assert size > 0 and lib.gpa_residual_norm_backward_workspace_bytes(4, 64, 3) == 0

    def bwd(dz=ok, z=ok, stats=ok, rows=4, gate=None, gate_rows=0, dx=ok, ws=ok, n=size):
        return lib.gpa_residual_norm_backward(dz, 64, ok, 64, z, 1, 64, ok, 1, 64, stats, gate, 1, gate_rows, rows,
                                              64, 0, None, None, 1, None, 1, dx, 64, ok, 64, None, None, None, None,
                                              None, ws, n, None)
    assert bwd(rows=0) == 1
    assert bwd(dz=odd) == 1 and bwd(z=None) == 1 and bwd(stats=None) == 1 and bwd(dx=None) == 1
    assert bwd(gate=ok, gate_rows=3) == 1
    assert bwd(ws=None) == 1 and bwd(n=size - 1) == 1 and b"workspace" in lib.gpa_last_error()


def test_workspace_covers_every_worker(lib):
    """One partial of five column sums per worker: never more workers than rows,
    at most about one per resident warp group."""
    for rows in (1, 2, 7, 1000, 274800):
        for cols in (8, 64, 264, 1024, 2048, 8192):
            for gate_rows in {rows, 1, rows // 2 or 1}:
                if rows % gate_rows:
                    continue
                n = lib.gpa_residual_norm_backward_workspace_bytes(rows, cols, gate_rows)
                workers, rest = divmod(n, 5 * cols * 4)
                assert rest == 0 and 1 <= workers <= min(rows, 2 * 148 * 16)


@pytest.mark.parametrize("name", ["x", "y", "gate", "weight", "bias", "post_weight", "post_bias"])
def test_forward_mode_derivatives_are_refused(name):
    from torch.autograd import forward_ad
    from gpa_vggt_b200 import kernels
    t = dict(x=_t(2, 16, dtype=F32), y=_t(2, 16, dtype=F32),
             **{k: _t(16, dtype=F32) for k in ("gate", "weight", "bias", "post_weight", "post_bias")})
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="CUDA device"):       # no tangent: refused for the CPU alone
            kernels.residual_norm(**t, post_kind="layer")
        t[name] = forward_ad.make_dual(t[name], torch.ones_like(t[name]))
        with pytest.raises(ValueError, match="residual_norm: no forward-mode"):
            kernels.residual_norm(**t, post_kind="layer")
