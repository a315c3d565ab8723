"""attention_shared_prefix refuses what it does not compute before anything is
launched (no GPU needed: shapes and types are checked before the device)."""
import ctypes
import pathlib
import subprocess
import sys

import pytest
import torch

ROOT = pathlib.Path(__file__).resolve().parents[1]
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def lib():
    from gpa_vggt_b200 import _lib, build
    build.build()
    return _lib.load()


def _args(R=2, H=4, M=3, D=64, Hk=2, P=5, N=7, dtype=BF16):
    def z(*s):
        return torch.zeros(*s, dtype=dtype)
    return [z(R, H, M, D), z(Hk, P, D), z(Hk, P, D), z(R, Hk, N, D), z(R, Hk, N, D), 0.125]


@pytest.mark.parametrize("error,change,kw", [
    (TypeError, dict(dtype=F32), {}),
    (ValueError, dict(D=96), {}),
    (ValueError, dict(H=3), {}),                                          # heads not a multiple of the key heads
    (ValueError, {}, dict(own_len=torch.zeros(3, dtype=torch.int32))),
    (TypeError, {}, dict(own_len=torch.zeros(2, dtype=torch.int64))),
    (TypeError, {}, dict(q_len=torch.zeros(2))),
    (ValueError, {}, dict(bias=torch.zeros(4))),
    (ValueError, {}, dict(bias=torch.zeros(4, 5))),                       # one row per query head
    (TypeError, {}, dict(bias=torch.zeros(5, dtype=torch.int32))),
    (ValueError, {}, dict(out=torch.zeros(2, 4, 3, 64))),                 # not bf16
    (ValueError, {}, dict(out=torch.zeros(2, 4, 4, 64, dtype=BF16))),
    (ValueError, {}, dict(out=torch.zeros(2, 4, 3, 68, dtype=BF16)[..., :64])),   # rows not 16-byte aligned
    (ValueError, {}, dict(out=torch.zeros(1, 4, 3, 64, dtype=BF16).expand(2, 4, 3, 64))),   # one row for two
    (ValueError, {}, dict(lse_out=torch.zeros(2, 1, 3).expand(2, 4, 3))),
    (ValueError, {}, dict(lse_out=torch.zeros(2, 4, 3, dtype=BF16))),
    (ValueError, {}, dict(lse_out=torch.zeros(2, 3, 4).transpose(1, 2))),
    (ValueError, {}, {}),                                                 # all well, but on the CPU
])
def test_refusals(error, change, kw):
    from gpa_vggt_b200 import kernels
    with pytest.raises(error, match="attention_shared_prefix"):
        kernels.attention_shared_prefix(*_args(**change), **kw)


@pytest.mark.parametrize("i,shape", [(0, (2, 4, 64)), (1, (2, 6, 64)), (2, (2, 5, 128)), (3, (3, 2, 7, 64)),
                                     (4, (2, 2, 8, 64)), (1, (1, 2, 5, 64))])
def test_shapes_that_do_not_fit(i, shape):
    from gpa_vggt_b200 import kernels
    args = _args()
    args[i] = torch.zeros(*shape, dtype=BF16)
    with pytest.raises(ValueError, match="attention_shared_prefix"):
        kernels.attention_shared_prefix(*args)


def test_gradients_are_refused():
    from gpa_vggt_b200 import kernels
    args = _args()
    args[1].requires_grad_(True)
    with pytest.raises(ValueError, match="no gradients"):
        kernels.attention_shared_prefix(*args)


def test_c_entry_refusals(lib):
    ok, odd = ctypes.c_void_p(256), ctypes.c_void_p(264)

    def run(q=ok, kp=ok, ko=ok, o=ok, R=2, M=3, H=4, Hk=2, D=64, P=5, N=7, stride=64, ws=ok, n=1 << 20):
        return lib.gpa_attention_shared_prefix(q, stride, 64, 64, kp, 64, 64, ok, 64, 64, None, 0, ko, 64, 64, 64,
                                               ok, 64, 64, 64, None, None, R, M, H, Hk, D, P, N, 0.125, 0, o, 64,
                                               64, 64, None, 0, 0, ws, n, None, None)
    assert run(R=0) == 0 and run(M=0) == 0                     # nothing to do
    assert run(R=-1) == 1 and run(H=3) == 1 and run(Hk=0) == 1 and run(P=-1) == 1 and run(N=-2) == 1
    assert run(D=32) == 3 and b"head_dim" in lib.gpa_last_error()
    assert run(R=1 << 20, M=1 << 12) == 3                      # 2^31 query rows
    assert run(P=(1 << 30) + 1) == 3
    assert run(q=None) == 1 and run(kp=None) == 1 and run(ko=None) == 1 and run(o=None) == 1
    assert run(q=odd) == 1 and run(kp=odd) == 1 and run(o=odd) == 1
    assert run(stride=60) == 1 and b"multiples of 8" in lib.gpa_last_error()
    assert run(ws=None) == 1 and run(ws=odd) == 1 and run(n=64) == 1 and b"workspace" in lib.gpa_last_error()


def test_workspace_size(lib):
    size = lib.gpa_attention_shared_prefix_workspace_bytes
    assert size(2, 3, 4, 3, 64, 5, 7) == -1 and size(2, 3, 4, 2, 96, 5, 7) == -1
    assert size(0, 3, 4, 2, 64, 5, 7) == 0 and size(2, 3, 4, 2, 64, 0, 0) == 0
    for R, M, H, Hk, D, P, N in [(1, 1, 1, 1, 64, 1, 0), (64, 1, 16, 16, 64, 66845, 1374), (4, 1374, 16, 16, 64, 16711, 1374),
                                 (5, 1, 16, 16, 64, 219840, 2748), (7, 45, 16, 2, 128, 5001, 777), (3, 515, 16, 8, 128, 4100, 1030)]:
        n = size(R, M, H, Hk, D, P, N)
        row = (D + 2) * 4                                      # a partial output, its maximum and sum
        assert n % row == 0 and n >= R * M * H * row
        assert n < 1 << 28


@pytest.mark.parametrize("heads", [128, 129, 256, 1000])
def test_more_query_heads_than_a_tile_has_rows(lib, heads):
    """One key head of more than 128 query heads: no whole token fits a 128-row tile."""
    code = ("from gpa_vggt_b200 import _lib; "
            f"print(_lib.load().gpa_attention_shared_prefix_workspace_bytes(2, 5, {heads}, 1, 64, 1000, 100))")
    got = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT)
    assert got.returncode == 0 and int(got.stdout.split()[-1]) >= 2 * 5 * heads * 66 * 4


def test_memory_that_is_written_is_not_read():
    from gpa_vggt_b200 import kernels
    args = _args()
    with pytest.raises(ValueError, match="outside the memory"):
        kernels.attention_shared_prefix(*args, out=args[0])
    big = torch.zeros(8 + 2 * 2 * 7 * 64, dtype=BF16)           # out begins eight values ahead of k_own
    args[3] = big[8:].view(2, 2, 7, 64)
    with pytest.raises(ValueError, match="outside the memory"):
        kernels.attention_shared_prefix(*args, out=big[:2 * 4 * 3 * 64].view(2, 4, 3, 64))
    both = torch.zeros(2 * 4 * 3 * 64, dtype=BF16)
    lse = both[:48].view(torch.float32).view(2, 4, 3)
    with pytest.raises(ValueError, match="outside the memory"):
        kernels.attention_shared_prefix(*_args(), out=both.view(2, 4, 3, 64), lse_out=lse)


def test_outputs_whose_rows_overlap():
    from gpa_vggt_b200 import kernels
    buf = torch.zeros(4096, dtype=BF16)
    with pytest.raises(ValueError, match="repeat rows"):
        kernels.attention_shared_prefix(*_args(), out=buf.as_strided((2, 4, 3, 64), (64, 192, 64, 1)))
    with pytest.raises(ValueError, match="CUDA device"):      # heads between the tokens: no overlap
        kernels.attention_shared_prefix(*_args(), out=buf[:1536].view(2, 3, 4, 64).transpose(1, 2))


@pytest.mark.parametrize("i", [1, 3])
def test_more_keys_than_an_index_holds(i):
    from gpa_vggt_b200 import kernels
    args = _args(R=1, Hk=1)
    for j in (i, i + 1):
        args[j] = torch.zeros(1, dtype=BF16).expand(*args[j].shape[:-2], 2 ** 32 + 5, 64)
    with pytest.raises(ValueError, match="2\\^30"):
        kernels.attention_shared_prefix(*args)


def test_status_word_of_another_type():
    from gpa_vggt_b200 import kernels
    with pytest.raises(ValueError, match="status"):
        kernels.attention_shared_prefix(*_args(), status=torch.zeros(1))


def test_strides_that_say_nothing():
    """A dim of one entry, or any dim of an empty tensor, may have any stride; the
    C entry takes multiples of 8 and must not see it."""
    from gpa_vggt_b200 import kernels
    odd = torch.zeros(2, 4 * 8 * 64 + 3, dtype=BF16)[:, :4 * 8 * 64].view(2, 4, 8, 64)[1:]
    first = torch.zeros(2 * 8 * 4 * 8 * 64, dtype=BF16)[:4 * 8 * 64].as_strided((1, 4, 8, 64), (7, 512, 64, 1))
    empty = torch.zeros(2, 2, 10, 68, dtype=BF16)[:, :, :0, :64]
    for t in (first, empty):
        assert t.is_contiguous()
        u, strides = kernels._vectors(t)
        assert u is t and not any(s % 8 for s in strides)
    assert odd.is_contiguous() and not any(s % 8 for s in kernels._vectors(odd)[1])   # (its base is odd: copied)


@pytest.mark.parametrize("i", [0, 1, 2, 3, 4, "bias"])
def test_forward_mode_derivatives_are_refused(i):
    from torch.autograd import forward_ad
    from gpa_vggt_b200 import kernels
    args, bias = _args(), torch.zeros(5)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="CUDA device"):       # no tangent: refused for the CPU alone
            kernels.attention_shared_prefix(*args, bias=bias)
        if i == "bias":
            bias = forward_ad.make_dual(bias, torch.ones(5))
        else:
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
        with pytest.raises(ValueError, match="attention_shared_prefix: no forward-mode"):
            kernels.attention_shared_prefix(*args, bias=bias)


def _call_bytes(lib, R, M, H, Hk, D, P, N, scale=0.125, q_sr=None):
    """Contiguous token-major queries and caches, a head-major prefix."""
    return lib.gpa_attention_shared_prefix_call_bytes(
        M * H * D if q_sr is None else q_sr, D, H * D, P * D, D, P * D, D, N * Hk * D, D, Hk * D, N * Hk * D, D, Hk * D,
        R, M, H, Hk, D, P, N, scale)


@pytest.mark.parametrize("size,folded", [((64, 1374, 16, 16, 64, 16711, 1374), False),
                                         ((200, 1374, 16, 16, 64, 66845, 1374), True),
                                         ((40, 3000, 16, 4, 128, 5000, 3000), False),
                                         ((8, 20000, 8, 8, 128, 0, 20000), False),
                                         ((1, 274800, 16, 16, 64, 66845, 0), False)])
def test_workspace_of_many_rows(lib, size, folded):
    """Only items that a span's end cuts leave parts, at most two to a CTA: 20 MB at
    head_dim 64, 39 at 128; beside them 8 bytes a row and part of its tile.  In a folded
    call with caches the few-rows kernel's outputs of the caches join in, one fp32 row
    of D + 2 values for each row (long calls cut no cache), and so every row tile of the
    prefix leaves its own: 4 D bytes a row twice, for 2 D of output."""
    R, M, H, Hk, D, P, N = size
    n = _call_bytes(lib, *size)
    out = R * M * H * D * 2
    rows = 128 * -(-M // (128 // (H // Hk))) * R * Hk
    copies = rows * 4 * D + R * M * H * 4 * (D + 2) if folded else 0
    assert 0 < n <= 148 * 2 * 2 * 128 * D * 4 + 3 * (8 * rows + 4 * R * Hk * M) + (1 << 16) + copies
    assert n < (40 << 20) + out // 4 + (copies if folded else 0)


def test_workspace_of_a_call(lib):
    """What a call takes is at most what any call of its sizes does, and less than that
    is refused; strides and scales that the tensor cores do not take count."""
    every = lib.gpa_attention_shared_prefix_workspace_bytes
    for size in [(1, 1, 1, 1, 64, 1, 0), (64, 1, 16, 16, 64, 66845, 1374), (4, 1374, 16, 16, 64, 16711, 1374),
                 (100, 1, 16, 16, 64, 9000, 33), (16, 17, 8, 8, 128, 9000, 90), (7, 45, 16, 2, 128, 5001, 777),
                 (3, 515, 16, 8, 128, 4100, 1030), (2, 300, 8, 1, 64, 0, 3000)]:
        R, M, H, Hk, D, P, N = size
        for kw in (dict(), dict(scale=-1.0), dict(q_sr=0), dict(q_sr=(M + 1) * H * D)):
            n = _call_bytes(lib, *size, **kw)
            assert 0 < n <= every(*size) and n % ((D + 2) * 4) == 0
    assert _call_bytes(lib, 2, 3, 4, 3, 64, 5, 7) == -1 and _call_bytes(lib, 2, 3, 4, 2, 96, 5, 7) == -1
    assert _call_bytes(lib, 0, 3, 4, 2, 64, 5, 7) == 0 and _call_bytes(lib, 2, 0, 4, 2, 64, 5, 7) == 0
    ok = ctypes.c_void_p(256)
    n = _call_bytes(lib, 4, 1374, 16, 16, 64, 16711, 1374)
    run = [ok, 1374 * 1024, 64, 1024, ok, 16711 * 64, 64, ok, 16711 * 64, 64, None, 0, ok, 1374 * 1024, 64, 1024, ok,
           1374 * 1024, 64, 1024, None, None, 4, 1374, 16, 16, 64, 16711, 1374, 0.125, 0, ok, 1374 * 1024, 64, 1024,
           None, 0, 0, ok, n - 16, None, None]
    assert lib.gpa_attention_shared_prefix(*run) == 1 and b"workspace" in lib.gpa_last_error()
