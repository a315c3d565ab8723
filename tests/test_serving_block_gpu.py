"""residual_norm and attention_shared_prefix as they are used together: streams
localised in a mapped scene (its merged K/V the prefix, the log counts the bias),
a frame of tokens and then token by token through a captured graph; and a stack of
gated residuals trained end to end.

Bounds: rel-L2 2e-2 against the same computation in 64 bits.  A value passes about
ten roundings to bf16 (2^-9 of it each, as a root mean square at most): 7e-3 if
they add up as independent ones, which projections and norms do not enlarge."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
BF16, F64 = torch.bfloat16, torch.float64


@pytest.fixture(scope="module", autouse=True)
def _build():
    from gpa_vggt_b200 import build
    build.build()


def rel(a, b):
    return float((a.double() - b).norm() / b.norm())


class Block:
    """Weights of one pre-norm block with LayerScale gates."""

    def __init__(self, C, H, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def rand(*s, scale=1.0, shift=0.0):
            return (torch.randn(*s, device="cuda", generator=g) * scale + shift).to(BF16)
        self.C, self.H, self.D = C, H, C // H
        self.qkv, self.proj = rand(3 * C, C, scale=C ** -0.5), rand(C, C, scale=C ** -0.5)
        self.fc1, self.fc2 = rand(2 * C, C, scale=C ** -0.5), rand(C, 2 * C, scale=(2 * C) ** -0.5)
        self.g1, self.g2 = rand(C, scale=0.2, shift=0.5), rand(C, scale=0.2, shift=0.5)
        self.n1, self.n2 = (rand(C, scale=0.1, shift=1.0), rand(C, scale=0.1)), (rand(C, scale=0.1, shift=1.0), rand(C, scale=0.1))
        self.n3 = (rand(C, scale=0.1, shift=1.0), rand(C, scale=0.1))


def block_kernels(b, x, h, caches, lens, prefix, bias, causal):
    """x, h = stream and its norm [R, M, C] -> the same after the block; appends to
    the caches at lens - M."""
    from gpa_vggt_b200 import kernels
    R, M, C = x.shape
    q, k, v = F.linear(h, b.qkv).view(R, M, 3, b.H, b.D).unbind(2)
    at = (lens[:, None] - M + torch.arange(M, device="cuda", dtype=torch.int32)).long()
    rows = torch.arange(R, device="cuda")[:, None]
    caches[0][rows, at], caches[1][rows, at] = k, v
    o = torch.empty(R, M, b.H, b.D, device="cuda", dtype=BF16)
    kernels.attention_shared_prefix(q.transpose(1, 2), prefix[0], prefix[1], caches[0].transpose(1, 2),
                                    caches[1].transpose(1, 2), b.D ** -0.5, own_len=lens, bias=bias, causal=causal,
                                    out=o.transpose(1, 2), status=torch.zeros(1, device="cuda", dtype=torch.int32))
    x, h = kernels.residual_norm(x, F.linear(o.view(R, M, C), b.proj), b.g1, *b.n2, 1e-6)
    return kernels.residual_norm(x, F.linear(F.gelu(F.linear(h, b.fc1)), b.fc2), b.g2, *b.n3, 1e-6)


def block_exact(b, x, h, caches, lens, prefix, bias, causal):
    d = lambda t: t.double()
    R, M, C = x.shape
    q, k, v = F.linear(h, d(b.qkv)).view(R, M, 3, b.H, b.D).unbind(2)
    outs = []
    for r in range(R):
        n = int(lens[r])
        caches[0][r, n - M:n], caches[1][r, n - M:n] = k[r], v[r]
        kk = torch.cat([d(prefix[0]), caches[0][r, :n].transpose(0, 1)], 1)
        vv = torch.cat([d(prefix[1]), caches[1][r, :n].transpose(0, 1)], 1)
        s = q[r].transpose(0, 1) @ kk.transpose(1, 2) * b.D ** -0.5
        s[..., :prefix[0].shape[1]] += d(bias)
        if causal:
            ahead = torch.arange(n, device="cuda")[None] > n - M + torch.arange(M, device="cuda")[:, None]
            s[..., prefix[0].shape[1]:].masked_fill_(ahead, -float("inf"))
        outs.append((s.softmax(-1) @ vv).transpose(0, 1).reshape(M, C))
    x = x + d(b.g1) * F.linear(torch.stack(outs), d(b.proj))
    h = F.layer_norm(x, (C,), d(b.n2[0]), d(b.n2[1]), 1e-6)
    x = x + d(b.g2) * F.linear(F.gelu(F.linear(h, d(b.fc1))), d(b.fc2))
    return x, F.layer_norm(x, (C,), d(b.n3[0]), d(b.n3[1]), 1e-6)


def merged_map(H, D, seed):
    """Merged keys, values and log counts of a three-frame scene."""
    from gpa_vggt_b200 import kernels
    from gpa_vggt_b200.merging.merge import build_plan
    g = torch.Generator().manual_seed(seed)
    S, w, h, ns = 3, 9, 9, 5
    N = S * (w * h + ns)
    metric = torch.randn(N, 256, generator=g).bfloat16().cuda()
    plan = build_plan(metric, w, h, 2, 2, int(N * 0.9), metric_dim=128, num_special=ns,
                      rand_idx=torch.randint(4, size=(S - 1, h // 2, w // 2), generator=g).cuda(),
                      proj=torch.randn(256, 128, generator=g).bfloat16().cuda())
    k, v = (torch.randn(H, N, D, generator=g).bfloat16().cuda() for _ in range(2))
    return (kernels.merge_kv(k, plan), kernels.merge_kv(v, plan)), plan.counts.log()


def test_streams_localised_in_a_map():
    """A chunk of tokens per stream of unequal lengths, then ten tokens one by one,
    replayed from one captured graph."""
    C, H, R, M, N = 512, 8, 4, 70, 160
    b = Block(C, H, 1)
    prefix, bias = merged_map(H, C // H, 2)
    g = torch.Generator(device="cuda").manual_seed(3)
    start = torch.tensor([0, 13, 60, 5], device="cuda", dtype=torch.int32)
    caches = [torch.randn(R, N, H, C // H, device="cuda", generator=g).to(BF16) for _ in range(2)]
    exact = [c.double() for c in caches]
    x = torch.randn(R, M, C, device="cuda", generator=g).to(BF16)
    h = F.layer_norm(x.float(), (C,), b.n1[0].float(), b.n1[1].float(), 1e-6).to(BF16)
    lens = start + M
    got = block_kernels(b, x, h, caches, lens, prefix, bias, True)
    want = block_exact(b, x.double(), h.double(), exact, lens, prefix, bias, True)
    assert rel(got[0], want[0]) < 2e-2 and rel(got[1], want[1]) < 2e-2

    token, norm = x[:, :1].clone(), h[:, :1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    spare = [c.clone() for c in caches]
    with torch.cuda.stream(side):
        block_kernels(b, token, norm, spare, lens + 1, prefix, bias, True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens += 1
        out = block_kernels(b, token, norm, caches, lens, prefix, bias, True)
    lens.copy_(start + M)
    for step in range(10):
        t = torch.randn(R, 1, C, device="cuda", generator=g).to(BF16)
        token.copy_(t)
        norm.copy_(F.layer_norm(t.float(), (C,), b.n1[0].float(), b.n1[1].float(), 1e-6))
        graph.replay()
        want = block_exact(b, token.double(), norm.double(), exact, lens, prefix, bias, True)
        assert rel(out[0], want[0]) < 2e-2 and rel(out[1], want[1]) < 2e-2
    assert lens.tolist() == (start + M + 10).tolist()


def test_a_stack_of_gated_residuals_learns_the_right_gradients():
    """Two modulated, normed sub-blocks as a fine-tuned head has them: the gradients
    of every leaf against differentiating the same stack in 64 bits."""
    from gpa_vggt_b200 import kernels
    g = torch.Generator(device="cuda").manual_seed(5)
    B, N, C = 3, 37, 256

    def leaf(*s, scale=1.0, shift=0.0):
        return (torch.randn(*s, device="cuda", generator=g) * scale + shift).requires_grad_(True)
    x, cond = leaf(B, N, C), leaf(B, 1, C)
    ws = [leaf(C, C, scale=C ** -0.5) for _ in range(2)]
    gates = [leaf(C, scale=0.3), leaf(C, C, scale=0.3 * C ** -0.5)]
    norms = [(leaf(C, scale=0.1, shift=1.0), leaf(C, scale=0.1)) for _ in range(3)]
    post = leaf(C, scale=0.1, shift=1.0)
    leaves = [x, cond, post, *ws, *gates, *(t for n in norms for t in n)]

    def stack(f, x, cond, post, w1, w2, g1, g2, a1, b1, a2, b2, a3, b3):
        z, h = f(x, x.new_zeros(()).expand_as(x), None, a1, b1, None)
        z, h = f(z, F.gelu(F.linear(h, w1)), g1, a2, b2, post)
        return f(z, torch.tanh(F.linear(h, w2)), F.linear(cond, g2), a3, b3, None)

    def fused(x, y, gate, w, b, post):
        return kernels.residual_norm(x, y.contiguous(), gate, w, b, 1e-6, post_kind=None if post is None else "rms",
                                     post_weight=post, post_eps=1e-6)

    def plain(x, y, gate, w, b, post):
        if post is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * post
        z = x + (y if gate is None else gate * y)
        return z, F.layer_norm(z, z.shape[-1:], w, b, 1e-6)
    dz, dh = (torch.randn(B, N, C, device="cuda", generator=g) for _ in range(2))
    got = torch.autograd.grad(stack(fused, *leaves), leaves, (dz, dh))
    exact = [t.detach().double().requires_grad_(True) for t in leaves]
    want = torch.autograd.grad(stack(plain, *exact), exact, (dz.double(), dh.double()))
    for a, b in zip(got, want):
        assert rel(a, b) < 1e-4          # fp32 throughout (TF32 is off): a few dozen operations of 2^-24, some cancelling
