"""Operator cases of the residual stream and of attention over a shared prefix.

Two operators, in the forms a transformer served and fine-tuned with this
package uses them:

* ``residual_norm``: z = x + gate * P(y) and h = N(z), the gated (and
  optionally post-normed) residual add of one sub-block with the norm in front
  of the next; ``residual_norm_train`` is the same with every gradient.
* ``shared_prefix``: softmax attention of a batch of requests over one set of
  prefix keys that all of them share (with a per-key bias, the log counts of
  merged keys) and each request's own cached keys.

With ``own`` false, ``run`` evaluates them with elementary torch operations in
32 bits; with ``own`` true it calls the package's operators.
"""
import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
TYPES = {"bf16": BF16, "fp32": F32}
LOG2E = 1.4426950408889634
EPS = 1e-6


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    def rn(name, op, batch, tokens, width, **kw):
        case = dict(name=name, op=op, batch=batch, tokens=tokens, width=width, stream="bf16", branch="bf16",
                    params="bf16", gate="channel", kind="layer", post="none")
        case.update(kw)
        return case

    def sp(name, requests, queries, heads, kv_heads, dim, prefix, cache, **kw):
        case = dict(name=name, op="shared_prefix", requests=requests, queries=queries, heads=heads,
                    kv_heads=kv_heads, dim=dim, prefix=prefix, cache=cache, bias=True, causal=False,
                    padded=False)
        case.update(kw)
        return case

    return [
        # the camera tokens of ten frames between two sub-blocks of the camera trunk: latency
        rn("norm 10x2048", "residual_norm", 1, 10, 2048),
        # one global block of 200 frames of 37x37 patches and 5 special tokens
        rn("norm 274800x1024", "residual_norm", 1, 274800, 1024),
        # a ragged batch with an fp32 stream, per-token gates and a normed branch
        rn("norm sandwich 4111x1536", "residual_norm", 3, 4111, 1536, stream="fp32", params="fp32",
           gate="token", kind="rms", post="rms"),
        # fine-tuning: a block over 20 frames, every gradient
        rn("train 27480x1024", "residual_norm_train", 1, 27480, 1024),
        # fine-tuning with an fp32 stream, one gate per sequence, normed branch, odd length
        rn("train sandwich 8x1375x768", "residual_norm_train", 8, 1375, 768, stream="fp32", params="fp32",
           gate="sequence", kind="layer", post="rms"),
        # one token of each of two streams against a four-frame map: latency
        sp("decode 2 requests", 2, 1, 16, 16, 64, 2361, 100),
        # one token of 64 streams against the merged keys of a 200-frame map
        sp("decode 64 requests", 64, 1, 16, 16, 64, 66845, 1374),
        # grouped heads of 128, no bias, long own caches
        sp("decode grouped 32 requests", 32, 1, 16, 4, 128, 8191, 4099, bias=False),
        # one token of 5 streams against the least merged keys of a 200-frame map
        sp("decode longest", 5, 1, 16, 16, 64, 219840, 2748),
        # a few tokens at a time, each after the other, ragged and padded
        sp("chunk 7 requests of 45", 7, 45, 16, 2, 128, 5001, 777, causal=True, padded=True),
        # a whole frame of tokens for each of 4 streams, over its own frame and the map
        sp("frames of 4 requests", 4, 1374, 16, 16, 64, 16711, 1374),
        # a longer chunk in order, grouped heads
        sp("chunk 3 requests of 515", 3, 515, 16, 8, 128, 4100, 1030, bias=False, causal=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["residual_norm", "residual_norm_train", "shared_prefix", "shared_prefix"])
    if op != "shared_prefix":
        train = op == "residual_norm_train"
        width = 8 * _log_int(rng, 8, 1024)
        batch = rng.randint(1, 9)
        most = (20000 * 1024 if train else 180000 * 1024) // (batch * width)
        tokens = _log_int(rng, 1, max(1, most))
        fp32 = rng.random() < 0.4
        if fp32:
            tokens = max(1, tokens // 3)
        return dict(op=op, batch=batch, tokens=tokens, width=width, stream="fp32" if fp32 else "bf16",
                    branch=rng.choice(["bf16", "fp32"]) if fp32 else "bf16", params="fp32" if fp32 else "bf16",
                    gate=rng.choice(["none", "channel", "sequence", "token"]), kind=rng.choice(["layer", "rms"]),
                    post=rng.choice(["none", "layer", "rms"]))
    heads, kv_heads = rng.choice([(16, 16), (16, 16), (16, 8), (16, 4), (12, 4), (8, 1), (15, 5)])
    dim = rng.choice([64, 64, 128])
    requests = _log_int(rng, 1, 64)
    queries = 1 if rng.random() < 0.5 else _log_int(rng, 2, 1374)
    most = 1_500_000_000 // (requests * queries * heads)     # scores of one pass
    cache = _log_int(rng, 1, max(1, min(4096, most // 2, 100_000 // requests)))
    prefix = 0 if rng.random() < 0.05 else _log_int(rng, 1, max(1, min(66845, most - cache)))
    return dict(op=op, requests=requests, queries=queries, heads=heads, kv_heads=kv_heads, dim=dim,
                prefix=prefix, cache=cache, bias=rng.random() < 0.6, causal=rng.random() < 0.4,
                padded=rng.random() < 0.3)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_attention(case, g) if case["op"] == "shared_prefix" else _prepare_norm(case, g)


def _prepare_norm(case, g):
    def rand(*shape, dtype, scale=1.0, shift=0.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(dtype)

    B, N, C = case["batch"], case["tokens"], case["width"]
    sd, bd, pd = (TYPES[case[k]] for k in ("stream", "branch", "params"))
    s = dict(case=case, x=rand(B, N, C, dtype=sd, scale=2.0, shift=0.3), y=rand(B, N, C, dtype=bd, scale=1.5))
    shape = {"none": None, "channel": (C,), "sequence": (B, 1, C), "token": (B, N, C)}[case["gate"]]
    # a gate of a trained LayerScale or of a modulation layer
    s["gate"] = None if shape is None else rand(*shape, dtype=pd, scale=0.3, shift=0.1)
    s["weight"] = rand(C, dtype=pd, scale=0.1, shift=1.0)
    s["bias"] = rand(C, dtype=pd, scale=0.1) if case["kind"] == "layer" else None
    s["post_weight"] = rand(C, dtype=pd, scale=0.1, shift=1.0) if case["post"] != "none" else None
    s["post_bias"] = rand(C, dtype=pd, scale=0.1) if case["post"] == "layer" else None
    if case["op"] == "residual_norm_train":
        s["dz"] = rand(B, N, C, dtype=sd, scale=0.5)
        s["dh"] = rand(B, N, C, dtype=bd, scale=0.7)
        for k in ("x", "y", "gate", "weight", "bias", "post_weight", "post_bias"):
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


def _prepare_attention(case, g):
    R, M, H, Hk, D = (case[k] for k in ("requests", "queries", "heads", "kv_heads", "dim"))
    P, N = case["prefix"], case["cache"]

    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=g).to(BF16)

    s = dict(case=case, scale=D ** -0.5)
    s["q"] = (1.5 * torch.randn(R, M, H, D, device="cuda", generator=g)).to(BF16).transpose(1, 2)
    # the shared prefix head-major, as the merge writes it; the caches token-major, as a projection fills them
    s["k_prefix"], s["v_prefix"] = rand(Hk, P, D), rand(Hk, P, D)
    s["k_own"], s["v_own"] = rand(R, N, Hk, D).transpose(1, 2), rand(R, N, Hk, D).transpose(1, 2)
    least = min(N, max(1, N // 4))
    s["own_len"] = torch.randint(least, N + 1, (R,), device="cuda", generator=g, dtype=torch.int32)
    s["own_len"][-1] = N
    s["q_len"] = None
    if case["padded"]:
        s["q_len"] = torch.randint(0, M + 1, (R,), device="cuda", generator=g, dtype=torch.int32)
        s["q_len"][0] = M
    # tokens behind each prefix key: mostly 1, a few of them merged from many
    counts = 1 + torch.floor(3 * torch.rand(P, device="cuda", generator=g) ** 8 * 8)
    s["bias"] = counts.log() if case["bias"] else None
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if op == "shared_prefix":
        return _own_attention(state) if own else _plain_attention(state)
    if op == "residual_norm":
        return _own_norm(state) if own else _plain_norm(state)
    return _own_norm_train(state) if own else _plain_norm_train(state)


def _own_norm(s):
    from gpa_vggt_b200 import kernels
    post = s["case"]["post"]
    z, h = kernels.residual_norm(s["x"], s["y"], s["gate"], s["weight"], s["bias"], EPS, kind=s["case"]["kind"],
                                 post_kind=None if post == "none" else post, post_weight=s["post_weight"],
                                 post_bias=s["post_bias"], post_eps=EPS)
    return {"z": z, "h": h}


def _own_norm_train(s):
    out = _own_norm(s)
    names = [k for k in ("x", "y", "gate", "weight", "bias", "post_weight", "post_bias") if s[k] is not None]
    grads = torch.autograd.grad((out["z"], out["h"]), [s[k] for k in names], (s["dz"], s["dh"]))
    return {"z": out["z"].detach(), "h": out["h"].detach(), **{"d" + k: v for k, v in zip(names, grads)}}


def _own_attention(s):
    from gpa_vggt_b200 import kernels
    out, lse = kernels.attention_shared_prefix(s["q"], s["k_prefix"], s["v_prefix"], s["k_own"], s["v_own"],
                                               s["scale"], own_len=s["own_len"], q_len=s["q_len"],
                                               bias=s["bias"], causal=s["case"]["causal"], return_lse=True)
    return {"out": out, "lse": lse}


def _normed(t, kind):
    """(normalised rows, 1/std) of fp32 rows."""
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    r = torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS)
    return t * r, r


def _normed_grad(d, n, r, kind):
    """Gradient of the rows from the gradient d of their normalised form n."""
    t = d - n * (d * n).mean(-1, keepdim=True)
    if kind == "layer":
        t = t - d.mean(-1, keepdim=True)
    return t * r


def _f(t):
    return None if t is None else t.detach().float()


def _plain_norm_values(s):
    c = s["case"]
    x, y, gate, w, b, pw, pb = (_f(s[k]) for k in ("x", "y", "gate", "weight", "bias", "post_weight", "post_bias"))
    yn = yr = None
    p = y
    if c["post"] != "none":
        yn, yr = _normed(y, c["post"])
        p = yn * pw if pb is None else yn * pw + pb
    z = x + p if gate is None else x + gate * p
    zn, zr = _normed(z, c["kind"])
    h = zn * w if b is None else zn * w + b
    return dict(p=p, yn=yn, yr=yr, z=z, zn=zn, zr=zr, h=h, gate=gate, w=w, pw=pw)


def _plain_norm(s):
    v = _plain_norm_values(s)
    return {"z": v["z"].to(s["x"].dtype), "h": v["h"].to(s["y"].dtype)}


def _plain_norm_train(s):
    c, v = s["case"], _plain_norm_values(s)
    dz, dh = s["dz"].float(), s["dh"].float()
    out = {"z": v["z"].to(s["x"].dtype), "h": v["h"].to(s["y"].dtype)}
    out["dweight"] = (dh * v["zn"]).sum((0, 1)).to(s["weight"].dtype)
    if s["bias"] is not None:
        out["dbias"] = dh.sum((0, 1)).to(s["bias"].dtype)
    d = dz + _normed_grad(dh * v["w"], v["zn"], v["zr"], c["kind"])
    out["dx"] = d.to(s["x"].dtype)
    dp = d
    if v["gate"] is not None:
        dg = d * v["p"]
        dg = {"channel": lambda: dg.sum((0, 1)), "sequence": lambda: dg.sum(1, keepdim=True),
              "token": lambda: dg}[c["gate"]]()
        out["dgate"] = dg.to(s["gate"].dtype)
        dp = d * v["gate"]
    if c["post"] != "none":
        out["dpost_weight"] = (dp * v["yn"]).sum((0, 1)).to(s["post_weight"].dtype)
        if s["post_bias"] is not None:
            out["dpost_bias"] = dp.sum((0, 1)).to(s["post_bias"].dtype)
        dp = _normed_grad(dp * v["pw"], v["yn"], v["yr"], c["post"])
    out["dy"] = dp.to(s["y"].dtype)
    return out


def _plain_attention(s):
    c = s["case"]
    R, M, H, Hk, D = (c[k] for k in ("requests", "queries", "heads", "kv_heads", "dim"))
    P, N, G = c["prefix"], c["cache"], H // Hk
    q = s["q"].float().reshape(R, Hk, G * M, D)
    kp, vp = s["k_prefix"].float(), s["v_prefix"].float()
    ko, vo = s["k_own"].float(), s["v_own"].float()
    # every request's queries over the shared keys in one product per head
    qp = q.transpose(0, 1).reshape(Hk, R * G * M, D)
    sp = (qp @ kp.transpose(1, 2)).view(Hk, R, G * M, P).transpose(0, 1) * s["scale"]
    if s["bias"] is not None:
        sp = sp + s["bias"]
    so = (q @ ko.transpose(2, 3)) * s["scale"]
    visible = _visible(s, R, M, N).repeat(1, G, 1)[:, None]                # [R, 1, G*M, N]
    scores = torch.cat([sp, so.masked_fill(~visible, -math.inf)], -1)
    del sp, so
    m = scores.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    scores = torch.exp(scores - m)
    l = scores.sum(-1, keepdim=True)
    pp = scores[..., :P].transpose(0, 1).reshape(Hk, R * G * M, P)
    o = (pp @ vp).view(Hk, R, G * M, D).transpose(0, 1) + scores[..., P:] @ torch.where(
        (torch.arange(N, device=q.device) < s["own_len"][:, None])[:, None, :, None], vo, torch.zeros_like(vo))
    o = torch.where(l > 0, o / l, torch.zeros_like(o)).reshape(R, H, M, D)
    lse = (m * LOG2E + torch.log2(l)).reshape(R, H, M)
    if s["q_len"] is not None:
        live = torch.arange(M, device=q.device) < s["q_len"][:, None]      # [R, M]
        o = torch.where(live[:, None, :, None], o, torch.zeros_like(o))
        lse = torch.where(live[:, None], lse, torch.full_like(lse, -math.inf))
    return {"out": o.to(BF16), "lse": lse}


def _visible(s, R, M, N):
    """[R, M, N]: which own keys each query sees."""
    keys, length = torch.arange(N, device="cuda"), s["own_len"].long()
    last = length[:, None].expand(R, M)
    if s["case"]["causal"]:
        queries = torch.full_like(length, M) if s["q_len"] is None else s["q_len"].long()
        last = torch.minimum(last, (length - queries)[:, None] + torch.arange(M, device="cuda") + 1)
    return keys < last[:, :, None]


# ---------------------------------------------------------------------------
# work and exact results
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "shared_prefix":
        R, M, H, Hk, D = (case[k] for k in ("requests", "queries", "heads", "kv_heads", "dim"))
        P, N = case["prefix"], case["cache"]
        # caches are filled between a quarter and the whole of their length, padded queries half on average
        n, m = 0.625 * N, M * (0.5 if case["padded"] else 1.0)
        pairs = R * H * m * (P + (n - m / 2 if case["causal"] and n > m else n))
        return {"bytes": 4.0 * Hk * D * (P + R * n) + (4.0 * P if case["bias"] else 0) + R * H * m * (4.0 * D + 4),
                "flops": 4.0 * D * pairs}
    rows, C = case["batch"] * case["tokens"], case["width"]
    sx, sy, sp = (4 if case[k] == "fp32" else 2 for k in ("stream", "branch", "params"))
    gates = {"none": 0, "channel": 1, "sequence": case["batch"], "token": rows}[case["gate"]]
    each = 2 * sx + 2 * sy
    if case["op"] == "residual_norm":
        return {"bytes": float(rows * C * each + gates * C * sp), "flops": 12.0 * rows * C}
    # forward, then dz, dh, x or z, and y again, and dx, dy out
    return {"bytes": float(rows * C * (each + 3 * sx + 3 * sy) + 3 * gates * C * sp), "flops": 40.0 * rows * C}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_attention(s) if case["op"] == "shared_prefix" else _exact_norm(s)


def _exact_norm(s):
    """The definition in 64 bits; gradients by differentiating it."""
    c = s["case"]
    names = ("x", "y", "gate", "weight", "bias", "post_weight", "post_bias")
    v = {k: None if s[k] is None else s[k].detach().double().requires_grad_(c["op"] == "residual_norm_train")
         for k in names}

    def norm(t, kind, w, b):
        mean = t.mean(-1, keepdim=True) if kind == "layer" else 0.0
        t = (t - mean) / torch.sqrt(((t - mean) ** 2).mean(-1, keepdim=True) + EPS)
        return t * w + (0.0 if b is None else b)

    u = v["y"] if c["post"] == "none" else norm(v["y"], c["post"], v["post_weight"], v["post_bias"])
    z = v["x"] + (u if v["gate"] is None else v["gate"] * u)
    h = norm(z, c["kind"], v["weight"], v["bias"])
    out = {"z": z.detach(), "h": h.detach()}
    if c["op"] == "residual_norm_train":
        given = [k for k in names if v[k] is not None]
        grads = torch.autograd.grad((z, h), [v[k] for k in given], (s["dz"].double(), s["dh"].double()))
        out.update({"d" + k: t for k, t in zip(given, grads)})
    return out


def _exact_attention(s):
    """The definition in 64 bits, one request and head at a time."""
    c = s["case"]
    R, M, H, Hk, D, N = (c[k] for k in ("requests", "queries", "heads", "kv_heads", "dim", "cache"))
    out = torch.zeros(R, H, M, D, device="cuda", dtype=F64)
    lse = torch.full((R, H, M), -math.inf, device="cuda", dtype=F64)
    lengths = s["own_len"].tolist()
    queries = [M] * R if s["q_len"] is None else s["q_len"].tolist()
    bias = 0.0 if s["bias"] is None else s["bias"].double()
    G = H // Hk
    for hk in range(Hk):
        kp, vp = s["k_prefix"][hk].double(), s["v_prefix"][hk].double()
        for r in range(R):
            n, m = lengths[r], queries[r]
            if m == 0:
                continue
            heads = slice(hk * G, hk * G + G)
            q = s["q"][r, heads, :m].double()                              # [G, m, D]
            own_scores = q @ s["k_own"][r, hk, :n].double().T * s["scale"]
            if c["causal"]:
                ahead = torch.arange(n, device="cuda")[None] - torch.arange(m, device="cuda")[:, None] > n - m
                own_scores = own_scores.masked_fill(ahead, -math.inf)
            scores = torch.cat([q @ kp.T * s["scale"] + bias, own_scores], -1)
            if scores.shape[-1] == 0:
                continue
            total = torch.logsumexp(scores, -1)
            p = torch.where(total[..., None] == -math.inf, 0.0, torch.exp(scores - total[..., None]))
            out[r, heads, :m] = p @ torch.cat([vp, s["v_own"][r, hk, :n].double()])
            lse[r, heads, :m] = total * LOG2E
    return {"out": out, "lse": lse}
