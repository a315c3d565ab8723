"""residual_norm against its formulas in 64 bits.

Bounds.  H is the largest relative error of one rounding to a type (half of its
eps).  z = round(x + round(gate * P(y))): two roundings.  h and the gradients are
compared with the formulas at z as kept, so they carry one rounding each plus
the fp32 arithmetic: a few operations per value, and for sums of n terms of any
sign at most depth * 2^-24 of the sum of their magnitudes, where depth, the
longest chain of additions, is below 256 here (a thread's terms, a row's or a
worker's, and the tree above them).  2^-16 of the magnitudes covers all of it.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
ARITH = 2.0 ** -16
EPS = 1e-6


@pytest.fixture(scope="module", autouse=True)
def _build():
    from gpa_vggt_b200 import build
    build.build()


def half(dtype):
    return torch.finfo(dtype).eps / 2


def near(got, ref, magnitude):
    """|got - ref| within one rounding to got's type and the arithmetic."""
    bound = half(got.dtype) * ref.abs() * 1.01 + ARITH * magnitude + 1e-30
    off = (got.double() - ref).abs() / bound
    assert bool((off <= 1).all()), float(off.max())


def make(shape, stream, branch, params, gate, kind, post, affine=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*s, dtype, scale=1.0, shift=0.0):
        return (torch.randn(*s, device="cuda", generator=g) * scale + shift).to(dtype)
    C = shape[-1]
    t = dict(x=rand(*shape, dtype=stream, scale=2, shift=0.3), y=rand(*shape, dtype=branch, scale=1.5))
    gs = {"none": None, "channel": (C,), "first": (shape[0],) + (1,) * (len(shape) - 2) + (C,), "token": shape}[gate]
    t["gate"] = None if gs is None else rand(*gs, dtype=params, scale=0.5, shift=0.1)
    for name, on in (("weight", kind), ("bias", kind == "layer"), ("post_weight", post),
                     ("post_bias", post == "layer")):
        w = name.endswith("weight")
        t[name] = rand(C, dtype=params, scale=0.2, shift=float(w)) if on and affine else None
    t["dz"], t["dh"] = rand(*shape, dtype=stream), rand(*shape, dtype=branch)
    return t


PARAMS = ("x", "y", "gate", "weight", "bias", "post_weight", "post_bias")


def norm64(t, kind, w, b):
    """(norm * w + b, the norm alone, 1/std)."""
    m = t.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(t[..., :1])
    r = ((t - m) ** 2).mean(-1, keepdim=True).add(EPS).rsqrt()
    n = (t - m) * r
    return n * (1 if w is None else w) + (0 if b is None else b), n, r


def norm64_grad(d, n, r, kind):
    """(gradient of the rows, a magnitude of its terms) from the gradient of the norm."""
    s1 = d.mean(-1, keepdim=True) if kind == "layer" else 0
    s2 = (d * n).mean(-1, keepdim=True)
    mag = r * (d.abs() + d.abs().mean(-1, keepdim=True) + n.abs() * (d * n).abs().mean(-1, keepdim=True))
    return r * (d - s1 - n * s2), mag


def column(t, shape):
    """Sum over the rows that share a gate row, in the gate's shape."""
    return t.sum_to_size(shape)


def check(t, kind, post, run):
    """run(t) -> z, h, {name: gradient}; every value against the formulas."""
    z, h, grads = run(t)
    v = {k: None if t[k] is None else t[k].detach().double() for k in PARAMS + ("dz", "dh")}
    x, y = v["x"], v["y"]
    if post:
        p, yn, yr = norm64(y, post, v["post_weight"], v["post_bias"])
        pmag = yn.abs() * (1 if v["post_weight"] is None else v["post_weight"].abs()) + (
            0 if v["post_bias"] is None else v["post_bias"].abs())
        # the mean is off by up to the arithmetic of the largest value
        pmag = pmag + yr * y.abs().amax(-1, keepdim=True)
    else:
        p, pmag = y, y.abs()
    gate = torch.ones((), device="cuda", dtype=F64) if v["gate"] is None else v["gate"]
    u = gate * p
    H = half(z.dtype)
    off = (z.double() - (x + u)).abs() / (1.01 * H * ((x + u).abs() + 2 * u.abs()) + ARITH * (x.abs() + gate.abs() * pmag))
    assert bool((off <= 1).all()), float(off.max())
    zk = z.detach().double()
    if kind:
        hr, zn, zr = norm64(zk, kind, v["weight"], v["bias"])
        w = torch.ones((), device="cuda", dtype=F64) if v["weight"] is None else v["weight"]
        spread = zr * zk.abs().amax(-1, keepdim=True)
        near(h, hr, w.abs() * (zn.abs() + spread) + (0 if v["bias"] is None else v["bias"].abs()))
    if grads is None:
        return
    d, dmag = v["dz"], v["dz"].abs()
    if kind:
        dn, nmag = norm64_grad(v["dh"] * w, zn, zr, kind)
        d, dmag = d + dn, dmag + nmag * (1 + spread)
        if "weight" in grads:
            near(grads["weight"], column(v["dh"] * zn, t["weight"].shape),
                 column((v["dh"] * (zn.abs() + spread)).abs(), t["weight"].shape))
        if "bias" in grads:
            near(grads["bias"], column(v["dh"], t["bias"].shape), column(v["dh"].abs(), t["bias"].shape))
    near(grads["x"], d, dmag)
    if "gate" in grads:
        near(grads["gate"], column(d * p, t["gate"].shape), column(dmag * pmag, t["gate"].shape))
    dp, dpmag = d * gate, dmag * gate.abs()
    if post:
        yspread = yr * y.abs().amax(-1, keepdim=True)
        if "post_weight" in grads:
            near(grads["post_weight"], column(dp * yn, t["post_weight"].shape),
                 column(dpmag * (yn.abs() + yspread), t["post_weight"].shape))
        if "post_bias" in grads:
            near(grads["post_bias"], column(dp, t["post_bias"].shape), column(dpmag, t["post_bias"].shape))
        pw = torch.ones((), device="cuda", dtype=F64) if v["post_weight"] is None else v["post_weight"]
        _, mag = norm64_grad(dpmag * pw.abs(), yn, yr, post)
        dp, dpmag = norm64_grad(dp * pw, yn, yr, post)[0], mag * (1 + yspread)
    near(grads["y"], dp, dpmag)


def call(t, kind, post, **kw):
    from gpa_vggt_b200 import kernels
    return kernels.residual_norm(t["x"], t["y"], t["gate"], t["weight"], t["bias"], EPS, kind=kind, post_kind=post,
                                 post_weight=t["post_weight"], post_bias=t["post_bias"], post_eps=EPS)


def forward(kind, post):
    def run(t):
        return (*call(t, kind, post), None)
    return run


def train(kind, post):
    def run(t):
        names = [k for k in PARAMS if t[k] is not None]
        for k in names:
            t[k] = t[k].detach().requires_grad_(True)
        z, h = call(t, kind, post)
        outs, given = ((z, h), (t["dz"], t["dh"])) if kind else ((z,), (t["dz"],))
        return z, h, dict(zip(names, torch.autograd.grad(outs, [t[k] for k in names], given)))
    return run


TYPES = [(BF16, BF16, BF16), (F32, BF16, F32), (F32, F32, F32), (BF16, BF16, F32)]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("kind,post,gate", [("layer", None, "channel"), ("rms", "rms", "first"),
                                            ("layer", "layer", "token"), (None, "layer", "none"),
                                            ("rms", None, "none"), (None, None, "token")])
@pytest.mark.parametrize("shape", [(3, 37, 1024), (1, 1, 8)])
def test_values_and_gradients(types, kind, post, gate, shape):
    check(make(shape, *types, gate, kind, post), kind, post, forward(kind, post))
    check(make(shape, *types, gate, kind, post), kind, post, train(kind, post))


@pytest.mark.parametrize("cols", [8, 40, 256, 264, 520, 768, 1032, 1536, 2048, 2056, 4096, 4104, 8192])
@pytest.mark.parametrize("post", [None, "rms"])
def test_every_width(cols, post):
    for types in TYPES[:3]:
        t = make((5, 13, cols), *types, "first", "layer", post, seed=cols)
        check(t, "layer", post, train("layer", post))


@pytest.mark.parametrize("shape,gate", [((4999, 256), "channel"), ((4999, 64), "token"), ((3000, 2, 64), "first"),
                                        ((2, 2500, 2048), "first"), ((1, 64), "channel"), ((700, 5, 1024), "first")])
def test_many_rows(shape, gate):
    """Rows split among the workers, and whole gate groups per worker."""
    t = make(shape, F32, BF16, F32, gate, "rms", "layer", seed=5)
    check(t, "rms", "layer", train("rms", "layer"))


def test_no_affine_and_part_of_the_parameters():
    t = make((2, 30, 512), F32, F32, F32, "channel", "layer", "rms", affine=False)
    check(t, "layer", "rms", train("layer", "rms"))
    t = make((2, 30, 512), BF16, BF16, BF16, "channel", "layer", "rms")
    t["bias"] = t["post_weight"] = None
    check(t, "layer", "rms", train("layer", "rms"))


def test_strided_rows_and_broadcast_inputs():
    g = torch.Generator(device="cuda").manual_seed(2)
    wide = torch.randn(6, 50, 3, 264, device="cuda", generator=g).bfloat16()
    t = make((6, 50, 264), BF16, BF16, BF16, "token", "layer", None)
    t["x"], t["y"] = wide[:, :, 0], wide[:, :, 2]              # rows of a wider buffer
    check(t, "layer", None, forward("layer", None))
    t["x"] = wide[:, :, 1, ::2].repeat(1, 1, 2)[..., :264].contiguous()[:, :, :264]
    t["y"] = wide.transpose(0, 1)[:6, :6, 0].repeat(1, 9, 1)[:, :50]   # rows in another order
    t["dz"] = torch.randn(6, 1, 264, device="cuda", generator=g).bfloat16().expand(6, 50, 264)
    check(t, "layer", None, train("layer", None))
    # a branch value shared by every token, and x also as the branch: their gradients add up
    y = torch.randn(6, 1, 264, device="cuda", generator=g, requires_grad=True)
    x = torch.randn(6, 50, 264, device="cuda", generator=g, requires_grad=True)
    from gpa_vggt_b200 import kernels
    z, h = kernels.residual_norm(x, y.expand(6, 50, 264), kind=None)
    gy, = torch.autograd.grad(z.sum(), y)
    assert torch.equal(gy, torch.full_like(gy, 50.0)) and h is None
    z, _ = kernels.residual_norm(x, x, kind=None)
    gx, = torch.autograd.grad(z, x, torch.ones_like(z))
    assert torch.equal(gx, torch.full_like(gx, 2.0))


def test_unaligned_base_is_copied():
    t = make((7, 64), BF16, BF16, BF16, "channel", "layer", None)
    for k in ("x", "y", "gate", "weight", "bias", "dz", "dh"):
        buf = torch.empty(t[k].numel() + 1, device="cuda", dtype=BF16)
        buf[1:] = t[k].reshape(-1)
        t[k] = buf[1:].view(t[k].shape)
    check(t, "layer", None, train("layer", None))


@pytest.mark.parametrize("used", ["z", "h"])
def test_one_output_unused(used):
    t = make((2, 9, 320), F32, F32, F32, "first", "layer", "layer")
    t["d" + ("h" if used == "z" else "z")].zero_()

    def run(t):
        names = [k for k in PARAMS if t[k] is not None]
        for k in names:
            t[k] = t[k].detach().requires_grad_(True)
        z, h = call(t, "layer", "layer")
        grads = torch.autograd.grad(z if used == "z" else h, [t[k] for k in names], t["d" + used])
        return z, h, dict(zip(names, grads))
    check(t, "layer", "layer", run)


def test_gradients_against_differences():
    """Central differences of a scalar of both outputs, in fp32 with a step of
    2^-6: they carry the third derivative times the step squared (below 1e-3 of
    the gradient's scale here) and 2^-24 / 2^-6 of the scalar's terms."""
    t = make((2, 3, 64), F32, F32, F32, "token", "layer", "rms")
    _, _, grads = train("layer", "rms")(t)

    def scalar():
        with torch.no_grad():
            z, h = call(t, "layer", "rms")
            return (z.double() * t["dz"]).sum() + (h.double() * t["dh"]).sum()
    step = 2.0 ** -6
    for name in PARAMS:
        if t[name] is None:
            continue
        flat, g = t[name].data.view(-1), grads[name].reshape(-1)
        for i in range(0, flat.numel(), max(1, flat.numel() // 11)):
            keep = flat[i].item()
            flat[i] = keep + step
            up = scalar()
            flat[i] = keep - step
            down = scalar()
            flat[i] = keep
            assert abs(float((up - down) / (2 * step)) - float(g[i])) < 5e-3 * (1 + float(grads[name].abs().max()))


def test_only_wanted_gradients_and_no_graph():
    from gpa_vggt_b200 import kernels
    t = make((4, 21, 512), BF16, BF16, BF16, "channel", "layer", None)
    z, h = call(t, "layer", None)
    assert not z.requires_grad and not h.requires_grad
    t["gate"].requires_grad_(True)
    with torch.no_grad():
        assert not call(t, "layer", None)[0].requires_grad
    z, h = call(t, "layer", None)
    (z.float().sum() + h.float().sum()).backward()
    assert t["gate"].grad is not None and t["x"].grad is None
    z, h = call(t, "layer", None)
    z.add_(1)                                       # z is kept for the gradients
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(h.float().sum(), t["gate"])
    assert kernels.residual_norm(t["x"][:0], t["y"][:0], t["gate"])[1].shape == (0, 21, 512)


def test_no_rows_have_zero_gradients():
    t = make((0, 7, 64), F32, BF16, F32, "channel", "layer", "layer")
    z, h, grads = train("layer", "layer")(t)
    assert z.shape == h.shape == (0, 7, 64)
    assert all(float(grads[k].abs().sum()) == 0 and grads[k].shape == t[k].shape for k in grads)


def test_infinities_and_nan_stay_in_their_rows():
    t = make((1, 40, 256), BF16, BF16, BF16, "channel", "layer", None)
    clean = call(t, "layer", None)
    t["y"][0, 3, 17], t["x"][0, 30, 5] = float("nan"), float("inf")
    z, h = call(t, "layer", None)
    rows = [r for r in range(40) if r not in (3, 30)]
    assert torch.equal(z[0, rows], clean[0][0, rows]) and torch.equal(h[0, rows], clean[1][0, rows])
    assert bool(torch.isnan(h[0, 3]).all()) and bool(torch.isnan(z[0, 3, 17])) and bool(torch.isinf(z[0, 30, 5]))


def test_same_bits_every_time_and_on_another_stream():
    run = train("layer", "rms")
    t = make((3, 900, 1024), BF16, BF16, BF16, "first", "layer", "rms")
    z, h, first = run(t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z2, h2, again = run(t)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(z, z2) and torch.equal(h, h2)
    assert all(torch.equal(first[k], again[k]) for k in first)


def test_captured_forward_and_backward_replay():
    """One training step captured into a CUDA graph: replays follow the inputs,
    and two graphs replayed in turn do not disturb each other."""
    def capture(seed):
        t = make((2, 130, 512), F32, BF16, F32, "first", "layer", "layer", seed=seed)
        run = train("layer", "layer")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            out = run(dict(t))
        torch.cuda.current_stream().wait_stream(s)
        del out
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(t)
        return t, g, out
    (ta, ga, oa), (tb, gb, ob) = capture(1), capture(2)
    with torch.no_grad():
        ta["x"].add_(0.5)
    for _ in range(2):
        ga.replay()
        gb.replay()
    torch.cuda.synchronize()
    check(ta, "layer", "layer", lambda _: oa)
    check(tb, "layer", "layer", lambda _: ob)


@pytest.mark.parametrize("cols", [256, 512, 1024, 2048])
def test_equals_the_two_kernels_it_replaces(cols):
    """residual_scale, then layernorm: the same bits."""
    from gpa_vggt_b200 import kernels
    for params in (BF16, F32):
        t = make((2, 687, cols), BF16, BF16, params, "channel", "layer", None)
        gate = t["gate"].bfloat16()
        z, h = kernels.residual_norm(t["x"], t["y"], gate, t["weight"], t["bias"], EPS)
        ref = kernels.residual_scale(t["x"], t["y"], gate)
        assert torch.equal(z, ref)
        assert torch.equal(h, kernels.layernorm(ref, t["weight"], t["bias"], EPS))


def test_block_calls_it_and_keeps_its_results(monkeypatch):
    from gpa_vggt_b200 import kernels
    from gpa_vggt_b200.vggt import layers
    torch.manual_seed(0)
    block = layers.Block(256, 4, init_values=0.3, qk_norm=True).cuda().bfloat16().eval()
    x = torch.randn(2, 77, 256, device="cuda").bfloat16()
    calls = []
    real = kernels.residual_norm
    monkeypatch.setattr(kernels, "residual_norm", lambda *a, **k: calls.append(1) or real(*a, **k))
    with torch.no_grad():
        out = block(x)
        y = layers._residual(x, block.ls1, block.attn(block.norm1(x)))
        ref = layers._residual(y, block.ls2, block.mlp(block.norm2(y)))
    assert calls == [1] and torch.equal(out, ref)


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_unused_norm_of_a_row_that_is_not_finite(kind):
    """With h unused, dx is dz for every row, as if there were no norm."""
    from gpa_vggt_b200 import kernels
    t = make((3, 5, 256), F32, BF16, BF16, "channel", kind, None)
    x = t["x"].detach().clone()
    x[1, 2, 7], x[2, 0, 9] = float("inf"), float("nan")
    x.requires_grad_(True)
    w = t["weight"].detach().clone().requires_grad_(True)
    z, _ = kernels.residual_norm(x, t["y"], t["gate"], w, None, EPS, kind=kind)
    dx, dw = torch.autograd.grad(z, [x, w], t["dz"])
    assert torch.equal(dx, t["dz"]) and not bool(dw.any())


@pytest.mark.parametrize("how", ["hook", "pre_hook", "instance", "subclass"])
def test_block_calls_a_norm_that_someone_watches(how):
    """Hooks on norm2, and forwards put in its place, run as they would without the fused pass."""
    from gpa_vggt_b200.vggt import layers
    torch.manual_seed(1)
    block = layers.Block(256, 4, init_values=0.3, qk_norm=True).cuda().bfloat16().eval()
    x = torch.randn(2, 33, 256, device="cuda").bfloat16()
    seen = []

    class Watched(layers.LayerNorm):
        def forward(self, x):
            seen.append(x.shape)
            return super().forward(x)

    with torch.no_grad():
        ref = block(x)
        if how == "hook":
            block.norm2.register_forward_hook(lambda m, i, o: seen.append(o.shape))
        elif how == "pre_hook":
            block.norm2.register_forward_pre_hook(lambda m, i: seen.append(i[0].shape))
        elif how == "instance":
            real = block.norm2.forward
            block.norm2.forward = lambda x: seen.append(x.shape) or real(x)
        else:
            block.norm2.__class__ = Watched
        out = block(x)
    assert seen == [x.shape] and torch.equal(out, ref)


def test_forward_mode_derivatives():
    """residual_norm refuses a dual tensor aloud; Block, whose kernels know no
    derivatives, keeps its values."""
    from torch.autograd import forward_ad
    from gpa_vggt_b200.vggt import layers
    t = make((2, 9, 256), BF16, BF16, BF16, "channel", "layer", None)
    torch.manual_seed(2)
    block = layers.Block(256, 4, init_values=0.3, qk_norm=True).cuda().bfloat16().eval()
    with torch.no_grad():
        ref = block(t["x"])
    with forward_ad.dual_level(), torch.no_grad():
        assert torch.equal(call(t, "layer", None)[0], call(t, "layer", None)[0])
        dual = forward_ad.make_dual(t["x"], torch.ones_like(t["x"]))
        assert torch.equal(forward_ad.unpack_dual(block(dual)).primal, ref)
        t["x"] = dual
        with pytest.raises(ValueError, match="forward-mode"):
            call(t, "layer", None)


def test_block_keeps_nothing_for_gradients():
    """Block's other bf16 kernels have no gradients, so no part of a graph is built
    (and no z, y and statistics kept) for it with gradients enabled."""
    from gpa_vggt_b200.vggt import layers
    torch.manual_seed(3)
    block = layers.Block(256, 4, init_values=0.3, qk_norm=True).cuda().bfloat16().eval()
    x = torch.randn(2, 33, 256, device="cuda").bfloat16()
    with torch.no_grad():
        ref = block(x)
    seen = []
    block.mlp.register_forward_pre_hook(lambda m, i: seen.append(i[0].requires_grad))
    out = block(x.requires_grad_(True))
    assert seen == [False] and not out.requires_grad and torch.equal(out, ref)


@pytest.mark.parametrize("shape", [(1, 256), (256, 1), (1, 1, 256), (1, 1, 1, 256)])
def test_block_with_a_gamma_of_more_dims(shape):
    """LayerScale's kernel takes any gamma of C values, and so does Block."""
    from gpa_vggt_b200.vggt import layers
    torch.manual_seed(4)
    block = layers.Block(256, 4, init_values=0.3, qk_norm=True).cuda().bfloat16().eval()
    x = torch.randn(2, 33, 256, device="cuda").bfloat16()
    with torch.no_grad():
        ref = block(x)
        block.ls1.gamma = torch.nn.Parameter(block.ls1.gamma.reshape(shape))
        assert torch.equal(block(x), ref)


def test_two_steps_at_once():
    """Training steps on two streams from two threads: the bits that each has alone."""
    import threading
    forms = [((3, 900, 1024), BF16, BF16, BF16, "first", "layer", None), ((7, 400, 264), F32, BF16, F32, "token", "rms", "layer"),
             ((1, 3000, 2048), F32, F32, F32, "channel", "layer", "rms")]
    cases = [(make(*f, seed=i), train(f[5], f[6])) for i, f in enumerate(forms)]
    want = [run(dict(t)) for t, run in cases]
    torch.cuda.synchronize()
    got = [[], []]

    def some(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(6):
                for t, run in cases:
                    got[i].append(run(dict(t)))
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=some, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for outs in got:
        assert len(outs) == 18
        for k, (z, h, grads) in enumerate(outs):
            wz, wh, wg = want[k % 3]
            assert torch.equal(z, wz) and torch.equal(h, wh) and all(torch.equal(grads[n], wg[n]) for n in wg)
