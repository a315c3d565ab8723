"""attention_shared_prefix against its definition in 64 bits.

Bounds.  H = 2^-8 is the largest relative error of a rounding to bf16.  The
probabilities are rounded to bf16 for the product with V: up to H * A, with
A = sum softmax * |v|; the output once more: H * |o|.  The arithmetic adds at
most 2^-10 * A: fp32 scores are off by up to D * 2^-23 * sum|q k| * scale (below
2^-13 for these inputs, and as much relative to a probability), and a chunk's
products with V are summed one after the other, a few thousand additions of
2^-23 each.  The log2 sums carry the scores' error, 2^-12, and the rounding of
the largest score.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
H8 = 2.0 ** -8
INF = float("inf")


@pytest.fixture(scope="module", autouse=True)
def _build():
    from gpa_vggt_b200 import build
    build.build()


def make(R, M, H, Hk, D, P, N, bias=None, own_len=None, q_len=None, causal=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*s, scale=1.0):
        return (torch.randn(*s, device="cuda", generator=g) * scale).to(BF16)
    a = dict(q=rand(R, H, M, D, scale=1.5), k_prefix=rand(Hk, P, D), v_prefix=rand(Hk, P, D),
             k_own=rand(R, Hk, N, D), v_own=rand(R, Hk, N, D), sm_scale=D ** -0.5, causal=causal,
             own_len=None, q_len=None, bias=None)
    if bias == "key":
        a["bias"] = torch.rand(P, device="cuda", generator=g) * 4
    elif bias == "head":
        a["bias"] = torch.randn(Hk, P, device="cuda", generator=g) * 2
    for name, v in (("own_len", own_len), ("q_len", q_len)):
        if v is not None:
            a[name] = torch.tensor(v, device="cuda", dtype=torch.int32)
    return a


def reference(a):
    """(o, sum softmax |v|, lse, largest |score|) in 64 bits, one request and query head at a time."""
    q = a["q"].double()
    R, H, M, D = q.shape
    Hk, P = a["k_prefix"].shape[:2]
    N = a["k_own"].shape[2]
    o = torch.zeros(R, H, M, D, device="cuda", dtype=F64)
    mag, lse = torch.zeros_like(o), torch.full((R, H, M), -INF, device="cuda", dtype=F64)
    top = torch.zeros(R, H, M, device="cuda", dtype=F64)
    lens = [N] * R if a["own_len"] is None else [min(max(v, 0), N) for v in a["own_len"].tolist()]
    qs = [M] * R if a["q_len"] is None else [min(max(v, 0), M) for v in a["q_len"].tolist()]
    for r in range(R):
        n, m = lens[r], qs[r]
        for h in range(H):
            hk = h // (H // Hk)
            keep = torch.ones(P, device="cuda", dtype=torch.bool)
            b = torch.zeros(P, device="cuda", dtype=F64)
            if a["bias"] is not None:
                b = (a["bias"] if a["bias"].dim() == 1 else a["bias"][hk if a["bias"].shape[0] > 1 else 0]).double()
                keep = b > -INF
            k = torch.cat([a["k_prefix"][hk, keep].double(), a["k_own"][r, hk, :n].double()])
            v = torch.cat([a["v_prefix"][hk, keep].double(), a["v_own"][r, hk, :n].double()])
            b = torch.cat([b[keep], torch.zeros(n, device="cuda", dtype=F64)])
            s = q[r, h, :m] @ k.T * a["sm_scale"] + b
            if a["causal"]:
                j = torch.arange(n, device="cuda")
                ahead = j[None] > (n - m) + torch.arange(m, device="cuda")[:, None]
                s[:, s.shape[1] - n:].masked_fill_(ahead, -INF)
            if s.shape[1] == 0 or m == 0:
                continue
            mx = s.amax(-1, keepdim=True)
            mx = torch.where(mx == -INF, torch.zeros_like(mx), mx)      # NaN stays
            e = torch.exp(s - mx)
            l = e.sum(-1, keepdim=True)
            some = l != 0
            p = torch.where(some, e / l, torch.zeros_like(e))
            o[r, h, :m], mag[r, h, :m] = p @ v, p @ v.abs()
            lse[r, h, :m] = torch.where(some, mx * math.log2(math.e) + torch.log2(l), torch.full_like(l, -INF))[:, 0]
            top[r, h, :m] = torch.where(s > -INF, s, torch.zeros_like(s)).abs().amax(-1)
    return o, mag, lse, top


def run(a, **kw):
    from gpa_vggt_b200 import kernels
    names = ("q", "k_prefix", "v_prefix", "k_own", "v_own", "sm_scale")
    return kernels.attention_shared_prefix(*(a[n] for n in names), own_len=a["own_len"], q_len=a["q_len"],
                                           bias=a["bias"], causal=a["causal"], return_lse=True, **kw)


def check(a, got=None):
    out, lse = run(a) if got is None else got
    o, mag, ref, top = reference(a)
    off = (out.double() - o).abs() / (H8 * (o.abs() + mag) + 2.0 ** -10 * mag + 1e-30)
    assert bool((off <= 1).all()), float(off.max())
    assert torch.equal(torch.isinf(lse), torch.isinf(ref)) and not bool(torch.isnan(lse).any())
    live = ~torch.isinf(ref)
    if bool(live.any()):
        off = (lse.double() - ref).abs()[live] / (2.0 ** -12 + 2.0 ** -21 * (top[live] + ref[live].abs()))
        assert bool((off <= 1).all()), float(off.max())
    return out, lse


SIZES = [
    # R, M, H, Hk, D, P, N
    (1, 1, 1, 1, 64, 1, 0),
    (1, 1, 1, 1, 64, 0, 1),
    (2, 1, 16, 16, 64, 130, 65),
    (3, 1, 4, 4, 128, 63, 64),
    (17, 1, 2, 2, 64, 1000, 33),            # more requests than a 16-row tile
    (70, 1, 3, 3, 64, 257, 9),              # more than a 64-row tile
    (5, 1, 16, 4, 64, 129, 300),            # grouped heads
    (2, 1, 15, 5, 128, 64, 1),
    (9, 1, 8, 1, 128, 700, 127),            # one key head
    (3, 7, 4, 2, 64, 128, 40),
    (2, 33, 6, 2, 64, 100, 90),
    (2, 50, 2, 2, 128, 65, 191),
    (1, 200, 2, 1, 64, 320, 200),
    (3, 130, 2, 2, 64, 200, 131),
    (2, 300, 4, 2, 128, 513, 310),
    (1, 600, 2, 2, 64, 1100, 700),
    (4, 129, 8, 2, 128, 0, 260),
    (2, 257, 3, 3, 64, 1025, 0),
    (40, 9, 2, 2, 64, 700, 50),             # few rows each, many together
    (150, 1, 3, 3, 128, 260, 5),
    (33, 2, 8, 2, 64, 129, 0),
    (20, 7, 6, 2, 128, 1500, 200),
]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("bias,causal", [(None, False), ("key", True), ("head", False)])
def test_sizes(size, bias, causal):
    check(make(*size, bias=bias, causal=causal, seed=sum(size)))


@pytest.mark.parametrize("size", [(6, 1, 4, 2, 64, 70, 300), (6, 60, 3, 3, 64, 500, 90), (6, 50, 2, 2, 128, 0, 90),
                                  (6, 5, 4, 4, 128, 70, 130), (6, 40, 2, 1, 64, 33, 200),
                                  (6, 140, 2, 1, 64, 300, 200), (6, 129, 2, 2, 128, 0, 140)])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(size, causal):
    """Own lengths from nothing to more than there is, shorter than the queries
    too; padded queries, none among them."""
    M, N = size[1], size[6]
    lens = [0, 1, N, N + 50, -3, N // 2 + 1]
    a = make(*size, bias="key", own_len=lens, q_len=[M, max(1, M // 2), M + 9, 0, M, 1], causal=causal, seed=3)
    # past a length a cache may hold anything
    for r, n in enumerate(lens):
        a["k_own"][r, :, max(n, 0):] = float("nan")
        a["v_own"][r, :, max(n, 0):] = INF
    check(a)


def test_no_keys_at_all():
    for M in (1, 20, 150):
        for P, N, lens in ((0, 0, None), (0, 70, [0, 0])):
            out, lse = run(make(2, M, 4, 2, 64, P, N, own_len=lens))
            assert float(out.abs().max()) == 0 and bool((lse == -INF).all())


@pytest.mark.parametrize("M", [1, 30, 300])
@pytest.mark.parametrize("D", [64, 128])
def test_masks_in_the_bias(M, D):
    """-inf takes keys out whatever they hold; the type's lowest value does not,
    so it alone still spreads a row evenly; large biases do not overflow."""
    a = make(2, M, 4, 2, D, 400, 0, bias="head", seed=1)
    out = torch.zeros(2, 400, device="cuda", dtype=torch.bool)
    out[0, ::3], out[1, 100:300], out[:, 399] = True, True, True
    a["bias"][out] = -INF
    a["k_prefix"][out], a["v_prefix"][out] = float("nan"), INF
    check(a)
    a["bias"][out] = float("nan")
    b = dict(a)
    b["bias"] = torch.where(out, -INF, a["bias"])
    check(b, run(a))
    a["bias"] = torch.full_like(a["bias"], -INF)
    o, lse = run(a)
    assert float(o.abs().max()) == 0 and bool((lse == -INF).all())
    a = make(2, M, 4, 2, D, 400, 0, bias="head", seed=2)
    low = torch.finfo(F32).min
    a["bias"].fill_(low)
    o, _ = run(a)
    mean = a["v_prefix"].double().mean(1).repeat_interleave(2, 0)[None, :, None]
    mag = a["v_prefix"].double().abs().mean(1).repeat_interleave(2, 0)[None, :, None]
    assert bool(((o.double() - mean).abs() <= H8 * (mean.abs() + mag) + 2.0 ** -10 * mag).all())
    a["bias"][:, ::2] = 3.0                 # beside others the lowest counts for nothing
    b = dict(a)
    b["bias"] = a["bias"].clone()
    b["bias"][:, 1::2] = -INF
    check(b, run(a))
    a["bias"] = (torch.arange(400, device="cuda") % 7).float() * 1000 - 3000
    check(a)


def test_large_scores():
    """Scores in the thousands: the running maximum carries them."""
    for M in (1, 20, 200):
        a = make(2, M, 4, 4, 64, 500, 200, seed=4)
        a["sm_scale"] = 30.0
        out, lse = run(a)
        o, mag, ref, top = reference(a)
        # scores up to 30 * sum|q k|: off by 64 * 2^-23 of it before the softmax
        slack = 64 * 2.0 ** -23 * 30 * 64 * 1.5 * 2
        assert bool(((out.double() - o).abs() <= (2 * H8 + 4 * slack) * (mag + 6)).all())
        assert bool(((lse.double() - ref).abs() <= slack * 2 + 2.0 ** -21 * ref.abs()).all())


def test_strided_views_and_in_place_buffers():
    g = torch.Generator(device="cuda").manual_seed(9)
    for M in (1, 19, 140):
        R, H, D, P, N = 3, 4, 64, 150, 90
        a = make(R, M, H, H, D, P, N, own_len=[90, 5, 44], seed=9)
        qkv = torch.randn(R, M, 3, H, D, device="cuda", generator=g).bfloat16()
        a["q"] = qkv[:, :, 0].transpose(1, 2)
        kv = torch.randn(R, N, 2, H, D, device="cuda", generator=g).bfloat16()
        a["k_own"], a["v_own"] = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
        rows = torch.randn(P, 2, H, D, device="cuda", generator=g).bfloat16()
        a["k_prefix"], a["v_prefix"] = rows[:, 0].transpose(0, 1), rows[:, 1].transpose(0, 1)
        a["bias"] = torch.rand(P, H, device="cuda", generator=g).t()              # not contiguous
        buf = torch.full((R, M + 2, H, D), 7.0, device="cuda", dtype=BF16)        # token-major, as proj reads it
        out = buf[:, 1:-1].transpose(1, 2)
        lse = torch.full((H, R, M), 5.0, device="cuda").transpose(0, 1)
        got = run(a, out=out, lse_out=lse)
        assert got[0].data_ptr() == out.data_ptr() and got[1].data_ptr() == lse.data_ptr()
        check(a, (out, lse))
        assert bool((buf[:, 0] == 7).all()) and bool((buf[:, -1] == 7).all())
        # bases and strides that vector loads cannot take are copied first
        odd = torch.randn(R * H * M * D + 1, device="cuda", generator=g).bfloat16()[1:].view(R, H, M, D)
        a["q"] = odd
        a["k_own"] = torch.randn(R, H, N, D + 4, device="cuda", generator=g).bfloat16()[..., :D]
        check(a)
        # one cache for every request, one key for every head
        a["k_own"] = a["k_own"][:1].expand(R, H, N, D)
        a["v_prefix"] = a["v_prefix"][:1].expand(H, P, D)
        check(a)


@pytest.mark.parametrize("size", [(3, 1, 2, 2, 64, 200, 50), (3, 30, 2, 2, 128, 200, 50), (3, 150, 2, 2, 64, 200, 50),
                                  (3, 150, 2, 2, 128, 200, 50), (30, 6, 2, 2, 64, 200, 50)])
def test_nan_and_infinity_of_keys_that_count(size):
    """A NaN or infinite score, in any key, makes its rows NaN and no others."""
    R = size[0]
    for key, value in [(0, float("nan")), (6, float("nan")), (7, INF), (13, -INF), (198, float("nan"))]:
        a = make(*size, seed=8)
        clean = run(a)
        a["k_own"][1, 1, key % 50, 3] = value
        a["k_prefix"][0, key, 5] = value
        out, lse = run(a)
        o, mag, ref, _ = reference(a)
        ok = torch.ones(R, 2, dtype=torch.bool, device="cuda")
        ok[:, 0] = False
        ok[1, 1] = False
        assert torch.equal(out[ok], clean[0][ok]) and torch.equal(lse[ok], clean[1][ok])
        bad = torch.isnan(ref)           # an infinite key gives -inf to half of the queries: they stay finite
        assert torch.equal(torch.isnan(lse), bad) and torch.equal(torch.isnan(out).any(-1), bad)
        assert bool(torch.isnan(out)[bad].all())


def test_values_that_are_not_finite():
    """A NaN in V reaches its feature of every row that sees the key."""
    for size in [(2, 1, 2, 2, 64, 200, 50), (2, 150, 2, 2, 128, 200, 50)]:
        a = make(*size, seed=8)
        clean, _ = run(a)
        a["v_prefix"][1, 77, 9] = float("nan")
        out, _ = run(a)
        assert bool(torch.isnan(out[:, 1, :, 9]).all())
        out[:, 1, :, 9] = clean[:, 1, :, 9]
        assert torch.equal(out, clean)


def test_queries_whose_requests_do_not_follow_on():
    """Requests further apart than their tokens, or queries shared by all."""
    for size in [(40, 4, 2, 2, 64, 300, 40), (3, 140, 2, 2, 128, 300, 40), (30, 1, 8, 1, 64, 300, 40)]:
        R, M, H, Hk, D = size[:5]
        a = make(*size, bias="key")
        wide = torch.zeros(R, M + 1, H, D, device="cuda", dtype=BF16)
        wide[:, :M] = a["q"].transpose(1, 2)
        a["q"] = wide[:, :M].transpose(1, 2)
        check(a)
        a["q"] = a["q"][:1].expand(R, H, M, D)
        check(a)


def test_scales():
    """Scales that are zero, negative or out of the ordinary."""
    for M in (1, 200):
        for scale in (0.0, -0.125, 1e-9, 1e-5):
            a = make(2, M, 2, 2, 64, 300, 100, bias="key", causal=True)
            a["sm_scale"] = scale
            check(a)


@pytest.mark.parametrize("M", [1, 40, 260])
def test_rows_past_q_len_are_left(M):
    a = make(3, M, 4, 2, 64, 100, 80, own_len=[80, 10, 3], q_len=[M, 0, max(M // 3, 1)], causal=True)
    out = torch.full((3, 4, M, 64), 3.0, device="cuda", dtype=BF16)
    lse = torch.full((3, 4, M), 11.0, device="cuda")
    run(a, out=out, lse_out=lse)
    live = (torch.arange(M, device="cuda")[None] < a["q_len"][:, None])[:, None].expand(3, 4, M)
    fresh, flse = check(a)
    assert torch.equal(out[live], fresh[live]) and torch.equal(lse[live], flse[live])
    assert bool((out[~live] == 3).all()) and bool((lse[~live] == 11).all())
    assert float(fresh[~live].abs().sum()) == 0 and bool((flse[~live] == -INF).all())


def test_offsets_past_32_bits():
    """Keys and values whose rows lie further apart than 2^31 elements."""
    step = (1 << 30) + 8
    buf = torch.zeros(4 * step + 64, device="cuda", dtype=BF16)
    for M in (1, 3, 150):
        a = make(2, M, 2, 2, 64, 5, 4, seed=6)
        far = torch.as_strided(buf, (1, 5, 64), (0, step, 1))
        far.copy_(a["k_prefix"][:1])
        a["k_prefix"] = far.expand(2, 5, 64)
        check(a)
        a["v_prefix"] = a["k_prefix"]
        own = torch.as_strided(buf, (1, 1, 4, 64), (0, 0, step, 1))
        a["k_own"] = own.expand(2, 2, 4, 64)
        a["v_own"] = torch.as_strided(buf, (2, 2, 4, 64), (2 * step, step, 0, 1))
        check(a)


def test_captured_call_follows_the_lengths():
    """A call captured into a graph reads the lengths, queries and caches of each
    replay; two graphs in turn do not disturb each other."""
    for M in (1, 50, 200):
        graphs = []
        for seed in (1, 2):
            a = make(4, M, 4, 2, 64, 300, 200, bias="key", own_len=[1, 2, 3, 4], causal=True, seed=seed)
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                _unchecked(a)
            torch.cuda.current_stream().wait_stream(s)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                got = _unchecked(a)
            graphs.append((g, a, got))
        for lens in ([200, 0, 77, 13], [64, 128, 5, 199]):
            for g, a, got in graphs:
                a["own_len"].copy_(torch.tensor(lens, dtype=torch.int32))
                a["q"].mul_(0.75)
                g.replay()
            for g, a, got in graphs:
                check(a, got)


def _unchecked(a):
    """run without reading the device status (which a capture cannot)."""
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    return run(a, status=status)


def test_same_bits_every_time_and_on_another_stream():
    for size in [(3, 1, 8, 2, 64, 5000, 777), (3, 300, 4, 2, 128, 900, 300)]:
        a = make(*size, bias="key", own_len=[5, size[6], 100])
        first = run(a)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            again = run(a)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_many_chunks():
    """A long prefix cut into many chunks, for few and for many rows."""
    check(make(1, 1, 2, 1, 64, 70000, 0, bias="key"))
    check(make(2, 140, 2, 2, 64, 30000, 150, bias="key"))
    check(make(1, 130, 1, 1, 128, 20001, 9000, causal=True))


@pytest.mark.parametrize("size", [
    (16, 17, 8, 8, 64, 9000, 90),       # folded: a pair of row tiles and one alone per head
    (16, 17, 8, 8, 128, 9000, 90),
    (100, 1, 16, 16, 64, 9000, 33),     # folded: one row tile, its keys in halves
    (30, 2, 16, 8, 128, 12000, 100),
    (2, 128, 8, 8, 64, 5000, 300),      # joint: one row tile each, in halves
    (3, 100, 4, 4, 128, 7000, 200),
    (5, 300, 4, 4, 64, 3000, 500),      # joint: pairs and one alone
    (3, 43, 6, 2, 64, 3000, 129),       # 126 rows a tile
    (1, 2000, 2, 1, 128, 1500, 1000),
])
def test_every_form_of_the_kernels(size):
    """Long enough for the tensor cores: items cut over many CTAs, odd tiles at the
    end, lengths and orders that leave parts of them empty."""
    R, M, N = size[0], size[1], size[6]
    g = torch.Generator().manual_seed(sum(size))
    lens = torch.randint(0, N + 1, (R,), generator=g).tolist()
    qs = torch.randint(0, M + 1, (R,), generator=g).tolist()
    check(make(*size, bias="key"))
    check(make(*size, own_len=lens, causal=True, seed=1))
    check(make(*size, bias="head", own_len=lens, q_len=qs, causal=bool(size[0] % 2), seed=2))
    a = make(*size, bias="key", own_len=[0] * R, seed=3)
    a["bias"][::5] = -INF
    a["k_prefix"][:, ::5] = float("nan")
    a["v_prefix"][:, ::5] = INF
    check(a)


def test_drawn_sizes():
    g = torch.Generator().manual_seed(77)

    def draw(lo, hi):
        return int(round(math.exp(float(torch.rand((), generator=g)) * math.log(hi / lo) + math.log(lo))))
    for i in range(40):
        H, Hk = [(4, 4), (8, 2), (6, 3), (5, 1)][int(torch.randint(4, (), generator=g))]
        R, M = draw(1, 40), draw(1, 400)
        P, N = draw(1, 6000), draw(1, 900)
        while R * M * H * (P + N) > 60_000_000:
            R, M = max(1, R // 2), max(1, M * 2 // 3)
            P = max(1, P // 2)
        lens = torch.randint(0, N + 1, (R,), generator=g).tolist()
        check(make(R, M, H, Hk, (64, 128)[i % 2], P, N, bias=(None, "key", "head")[i % 3], own_len=lens,
                   q_len=torch.randint(0, M + 1, (R,), generator=g).tolist() if i % 4 == 0 else None,
                   causal=i % 5 < 2, seed=i))


def test_equals_attention_over_the_joined_keys():
    """The same softmax as kernels.attention over prefix and own keys in a row."""
    from gpa_vggt_b200 import kernels
    a = make(3, 200, 4, 4, 64, 300, 100, bias="head")
    o, lse = run(a)
    k = torch.cat([a["k_prefix"].expand(3, 4, 300, 64), a["k_own"]], 2)
    v = torch.cat([a["v_prefix"].expand(3, 4, 300, 64), a["v_own"]], 2)
    b = torch.cat([a["bias"], torch.zeros(4, 100, device="cuda")], 1)[None].expand(3, 4, 400)
    ro, rl = kernels.attention(a["q"], k, v, b, a["sm_scale"], return_lse=True)
    mag = reference(a)[1]
    assert bool(((o.double() - ro.double()).abs() <= 2 * (2 * H8 + 2.0 ** -10) * mag).all())
    # attention adds the bias as a pair of bf16: 2^-16 of it
    assert float((lse - rl).abs().max()) < 2.0 ** -11 + 2.0 ** -13


def test_public_form_casts_as_attention_keybias():
    from gpa_vggt_b200.merging import attention_shared_prefix
    a = make(2, 30, 4, 2, 64, 90, 40, bias="key", own_len=[40, 7], causal=True)
    a["bias"] = a["bias"].bfloat16().float()
    f = {k: v.float() if torch.is_tensor(v) and v.dtype == BF16 else v for k, v in a.items()}
    got = attention_shared_prefix(f["q"], f["k_prefix"], f["v_prefix"], f["k_own"], f["v_own"], f["bias"],
                                  f["sm_scale"], own_len=f["own_len"], causal=True, return_lse=True)
    want = run(a)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(NotImplementedError):
        attention_shared_prefix(*(f[k].half() for k in ("q", "k_prefix", "v_prefix", "k_own", "v_own")), None, 0.1)


@pytest.mark.parametrize("size", [(2, 1, 129, 1, 64, 300, 40), (1, 3, 256, 1, 128, 130, 70), (2, 2, 400, 2, 64, 0, 65)])
def test_more_query_heads_than_a_tile_has_rows(size):
    check(make(*size, bias="key", own_len=[size[-1], 3][:size[0]], causal=True, seed=4))


@pytest.mark.parametrize("size,own_len", [
    ((1, 1, 1, 1, 64, 20000, 0), None),            # more than 128 chunks of a row
    ((2, 1, 1, 1, 128, 20000, 90), [90, 0]),
    ((2, 1, 4, 4, 64, 9000, 70), [0, 70]),         # more than 32
    ((4, 12, 16, 4, 64, 0, 1500), [1500, 0, 3, 700]),   # four warps a row
    ((18, 2, 32, 16, 64, 1288, 54), None),         # two
    ((8, 64, 16, 16, 64, 0, 700), [700, 64, 0, 1, 699, 300, 65, 10]),   # one, of many rows
    ((3, 40, 16, 2, 128, 2500, 200), [200, 0, 41]),     # few row tiles in many parts
])
def test_every_width_of_the_join(size, own_len):
    check(make(*size, bias="key" if size[5] else None, own_len=own_len, causal=True, seed=6))


@pytest.mark.parametrize("M", [1, 300])
def test_strides_that_say_nothing(M):
    """One request, and no prefix or cache at all, cut out of buffers whose rows lie an
    odd number of values apart."""
    a = make(1, M, 4, 2, 64, 3000, 200, bias="key", seed=12)
    g = torch.Generator(device="cuda").manual_seed(13)

    def odd(t):
        buf = torch.randn(t.numel() + 16, device="cuda", generator=g).bfloat16()[:t.numel()]
        view = buf.as_strided(t.shape, (t.numel() + 3, *t.stride()[1:]))
        view.copy_(t)
        return view
    for name in ("q", "k_own", "v_own"):
        a[name] = odd(a[name])
        assert a[name].stride(0) % 8 and a[name].is_contiguous()
    out = odd(torch.zeros(1, 4, M, 64, device="cuda", dtype=BF16))
    got = run(a, out=out)
    check(a, got)
    wide = torch.zeros(1, 2, 200, 68, device="cuda", dtype=BF16)[:, :, :0, :64]
    a["k_own"], a["v_own"] = wide, wide
    check(a)
    a = make(1, M, 4, 2, 64, 0, 200, seed=12)
    a["k_prefix"], a["v_prefix"] = wide[0], wide[0]
    check(a)


EVERY_KERNEL = [                        # sizes at which each kernel, and each form of it, runs
    (2, 1, 4, 2, 64, 700, 40), (3, 30, 2, 2, 128, 700, 40),
    (5, 300, 4, 4, 64, 3000, 500), (3, 260, 4, 4, 128, 3000, 500),       # joint, pairs of row tiles
    (2, 128, 8, 8, 64, 5000, 300), (3, 100, 4, 4, 128, 7000, 200),       # joint, in halves
    (16, 17, 8, 8, 64, 9000, 90), (100, 1, 16, 16, 64, 9000, 33),        # folded
]


@pytest.mark.parametrize("size", EVERY_KERNEL)
def test_large_biases(size):
    """The largest bias wins, however large: a row is its key's value, whichever kernel
    runs.  Beyond 1e30 biases are alike."""
    R, Hk, P = size[0], size[3], size[5]
    g = torch.Generator(device="cuda").manual_seed(21)

    def best(a, k, v):
        """Key k of a head's prefix alone counts; its bias is v."""
        out, lse = run(a)
        want = torch.stack([a["v_prefix"][i, k[i]] for i in range(Hk)]).repeat_interleave(size[2] // Hk, 0)
        assert torch.equal(out, want[None, :, None].expand_as(out))
        # a bias is rounded to fp32 (on the tensor cores over the scale), and the score with it
        assert bool(((lse.double() - v * math.log2(math.e)).abs() <= 2.0 ** -21 * abs(v) * math.log2(math.e)).all())

    for low, high, own in [(1e9, 2e9, None), (1e6, 4e9, None), (-2e9, -1e9, 0), (-1e30, -1e12, 0), (1e29, 9e29, None)]:
        for place in (0, P // 2, P - 1):
            a = make(*size, bias="head", own_len=None if own is None else [own] * R, seed=22)
            k = [(place + 131 * i) % P for i in range(Hk)]
            a["bias"] = low * (1 + torch.rand(Hk, P, device="cuda", generator=g) / (4 if low > 0 else -4))
            a["bias"][torch.arange(Hk), k] = high
            best(a, k, high)
    for side in (1, -1):
        a = make(*size, bias="head", own_len=[0] * R, seed=23)
        a["bias"].fill_(-INF)
        top = torch.tensor([1e31, 1e30, torch.finfo(F32).max, 5e33], device="cuda") * side
        a["bias"][:, [3, P // 2, P - 2, P - 1]] = top
        out, _ = run(a)
        v = a["v_prefix"][:, [3, P // 2, P - 2, P - 1]].double().repeat_interleave(size[2] // Hk, 0)
        mean, mag = v.mean(1)[None, :, None], v.abs().mean(1)[None, :, None]
        assert bool(((out.double() - mean).abs() <= H8 * (mean.abs() + mag) + 2.0 ** -10 * mag).all())


@pytest.mark.parametrize("size", EVERY_KERNEL)
@pytest.mark.parametrize("scale", [0.125, 16.0])
def test_exact_scores_that_move_the_maximum(size, scale):
    """Small whole numbers in q and k: the scores, up to some thousands, are exact in
    fp32, so the ordinary bounds hold; later keys score higher, so the maximum moves
    often, and the first keys are out, so rows begin without one."""
    R, M, H, Hk, D, P, N = size
    g = torch.Generator(device="cuda").manual_seed(31)

    def whole(*s):
        return torch.randint(-1, 2, s, device="cuda", generator=g).to(BF16)
    for causal in (False, True):
        a = make(*size, bias="head", own_len=[(37 * r) % (N + 1) for r in range(R)], causal=causal, seed=32)
        a["sm_scale"] = scale
        a["q"] = whole(R, H, M, D)
        for name, n in (("k_prefix", P), ("k_own", N)):
            grow = 1 + 6 * torch.arange(n, device="cuda")[:, None] // n
            a[name] = whole(*a[name].shape) * grow.to(BF16)
        a["bias"] = torch.randint(0, 4, (Hk, P), device="cuda", generator=g).float() * scale
        a["bias"][:, :P // 3] = -INF
        check(a)
        a["bias"].fill_(-INF)                   # the caches alone, some of them empty
        check(a)


@pytest.mark.parametrize("size", EVERY_KERNEL + [(7, 45, 16, 2, 128, 5001, 777), (40, 9, 16, 16, 64, 30000, 600)])
def test_whatever_the_workspace_holds(size):
    """Nothing of a workspace is read before the call has written it."""
    R, M, N = size[0], size[1], size[6]
    a = make(*size, bias="key", own_len=[(91 * r) % (N + 1) for r in range(R)],
             q_len=[(53 * r + M) % (M + 1) for r in range(R)], causal=True, seed=41)
    want = run(a)
    for value in (float("nan"), 3.0e38, -1.0):
        torch.cuda.synchronize()
        held = [torch.full((1 << n,), value, device="cuda") for n in range(10, 25)]
        del held                               # the allocator hands it to the call
        got = run(a)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_memory_of_a_large_call():
    """64 frames of 1,374 tokens: 180 MB of output, and beside it what the cut items
    leave (20 MB) and 24 bytes a row, not copies of every row."""
    a = make(64, 1374, 16, 16, 64, 2000, 300, seed=42)
    _unchecked(a)
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out, lse = _unchecked(a)
    used = torch.cuda.max_memory_allocated() - before - out.numel() * 2 - lse.numel() * 4
    assert used < 64 << 20, used
    r, h = 63, 15                               # the last rows, against the same request alone
    one = {k: v[r:r + 1] if k in ("q", "k_own", "v_own") else v for k, v in a.items()}
    ref = reference({**one, "q": one["q"][:, h:], "k_prefix": a["k_prefix"][h:], "v_prefix": a["v_prefix"][h:],
                     "k_own": one["k_own"][:, h:], "v_own": one["v_own"][:, h:]})
    off = (out[r:, h:].double() - ref[0]).abs() / (H8 * (ref[0].abs() + ref[1]) + 2.0 ** -10 * ref[1] + 1e-30)
    assert bool((off <= 1).all())


@pytest.mark.parametrize("size", EVERY_KERNEL)
def test_accuracy_of_the_sums(size):
    """Rows of two keys with exact scores, the second up to 2^8 times the first, on every
    lane of a tile: the log2 sum is within 2^-13, more than log2(1 + 7.7e-5) = 1.11e-4
    of the cubic, and a few roundings of sums below 16."""
    R, M, H, Hk, D, P, N = size
    g = torch.Generator(device="cuda").manual_seed(51)
    for j in list(range(128, 136)) + [3, 255]:
        a = make(*size, bias="key", own_len=[0] * R, seed=52)
        a["q"].zero_()
        a["q"][..., 0] = (torch.rand(R, H, M, device="cuda", generator=g) * 44).bfloat16()
        a["k_prefix"].zero_()
        a["k_prefix"][:, j, 0] = 1
        a["sm_scale"] = 0.125
        a["bias"].fill_(-INF)
        a["bias"][[0, j]] = 0
        _, lse = run(a)
        ref = torch.log2(1 + torch.exp(a["q"][..., 0].double() * 0.125))
        assert float((lse.double() - ref).abs().max()) <= 2.0 ** -13 + 2.0 ** -20


def test_two_calls_at_once():
    """Calls of every kernel on two streams with nothing between them, and from two
    threads: each has its own workspace, and the bits it has alone."""
    import threading
    cases = [make(*size, bias="key", own_len=[size[6] // (r + 1) for r in range(size[0])], causal=True, seed=61 + i)
             for i, size in enumerate(EVERY_KERNEL)]
    want = [run(a) for a in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]

    def some(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(3):
                for a in cases[::-1] if i else cases:
                    got[i].append(_unchecked(a))

    for _ in range(2):                          # interleaved by hand, then by the threads
        for a, b in zip(cases, cases[::-1]):
            for i, c in ((0, a), (1, b)):
                with torch.cuda.stream(streams[i]):
                    got[i].append(_unchecked(c))
    threads = [threading.Thread(target=some, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        assert len(outs) == 5 * len(cases)
        for k, (o, lse) in enumerate(outs):
            w = want[::-1][k % len(cases)] if i else want[k % len(cases)]
            assert torch.equal(o, w[0]) and torch.equal(lse, w[1])


@pytest.mark.parametrize("M", [1, 260])
@pytest.mark.parametrize("dtype", [torch.float16, BF16, F32, F64])
def test_lowest_bias_of_every_type(M, dtype):
    """A row of nothing but the type's lowest value spreads evenly; beside another key
    it counts for nothing, and -inf (or NaN) takes a key out."""
    a = make(3, M, 4, 4, 64, 3000, 40, own_len=[0] * 3, seed=71)
    a["q"].zero_()
    a["bias"] = torch.full((4, 3000), torch.finfo(dtype).min, device="cuda", dtype=dtype)
    o, lse = run(a)
    v = a["v_prefix"].double()
    mean, mag = v.mean(1)[None, :, None], v.abs().mean(1)[None, :, None]
    assert bool(((o.double() - mean).abs() <= H8 * (mean.abs() + mag) + 2.0 ** -10 * mag).all())
    assert bool(torch.isfinite(lse).all())
    a["bias"][:, 1000:] = -INF
    a["bias"][:, 1500] = float("nan")
    a["bias"][:, 77] = torch.finfo(dtype).max if dtype != torch.float16 else 0
    o, _ = run(a)
    assert torch.equal(o, a["v_prefix"][:, 77][None, :, None].expand_as(o))


def test_public_form_keeps_the_lowest_bias_finite():
    """fp32's lowest value stays a weight when the public form casts to bf16."""
    from gpa_vggt_b200.merging import attention_shared_prefix
    a = make(2, 5, 4, 2, 64, 90, 40, own_len=[0, 0])
    a["q"].zero_()
    f = {k: a[k].float() for k in ("q", "k_prefix", "v_prefix", "k_own", "v_own")}
    bias = torch.full((90,), torch.finfo(F32).min, device="cuda")
    bias[30:] = -INF
    o = attention_shared_prefix(*f.values(), bias, 0.125, own_len=a["own_len"])
    v = a["v_prefix"][:, :30].double().repeat_interleave(2, 0)
    mean, mag = v.mean(1)[None, :, None], v.abs().mean(1)[None, :, None]
    assert bool(((o.double() - mean).abs() <= H8 * (mean.abs() + mag) + 2.0 ** -10 * mag).all())
