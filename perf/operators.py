"""The operators around a hyper-connection layer's block, measured.

Four operators, each in its plain form (elementary torch operations in 32 bits,
rounded once at the end) and, where ``own`` is true, as calls of
``hyperconnections_b200.ops``:

* ``hc_read_norm``: the width-read u = R x of n streams and the block's
  pre-norm over the m D values of u;
* ``hc_mix_write_norm``: the block's post-norm, gate, residual scale and
  dropout, then the mix H x and the depth-write W z into the n streams;
* ``hc_dropout``: dropout whose mask comes from a counter-based generator
  (Philox 4x32-10 of Salmon, Moraes, Dror and Shaw, 2011) and is never stored;
* ``gated_ffn``: y = (act(x Wg^T) * (x Wu^T)) Wd^T.

A "serve" case is the forward pass alone, a "train" case the forward and the
backward pass with every gradient. Sizes are those of this repository's
benchmark (n = 4 streams, 16,384 tokens of D = 768), of its ViT (D = 384) and
decoder LM (D = 2048, hidden 8192), of its n x D sweep, and odd ones.
"""

from __future__ import annotations

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# --------------------------------------------------------------------- cases
def listed():
    return [
        # one decoding step of the LM for eight sequences: latency
        dict(name="read_norm_decode", op="read_norm", mode="serve", type="bf16", T=8, n=4, m=1, D=2048, norm="rms", bias=False),
        # the benchmark's 16,384 tokens through a pre-norm, forward and backward
        dict(name="read_norm_train", op="read_norm", mode="train", type="bf16", T=16384, n=4, m=1, D=768, norm="rms", bias=False),
        # two backbone blocks, LayerNorm, a row length no vector divides, float32 streams
        dict(name="read_norm_odd", op="read_norm", mode="train", type="fp32", T=1003, n=3, m=2, D=333, norm="layer", bias=True),
        # the block's output written back in the same decoding step
        dict(name="write_norm_decode", op="write_norm", mode="serve", type="bf16", T=8, n=4, m=1, D=2048, norm="rms", bias=False,
             gate="sigmoid", scale=True, proj=False, p=0.0),
        # the benchmark's tokens: post-norm, sigmoid gate, layer scale, dropout
        dict(name="write_norm_train", op="write_norm", mode="train", type="bf16", T=16384, n=4, m=1, D=768, norm="rms", bias=False,
             gate="sigmoid", scale=True, proj=False, p=0.1),
        # the sweep's n = 8 with two blocks, LayerNorm, the projected mix, fp16
        dict(name="write_norm_wide", op="write_norm", mode="train", type="fp16", T=4096, n=8, m=2, D=1024, norm="layer", bias=True,
             gate="", scale=True, proj=True, p=0.0),
        # the embedding of a small batch of the ViT: 8 images of 64 patches
        dict(name="dropout_small", op="dropout", mode="train", type="fp16", N=8 * 64 * 384 + 5, p=0.1),
        # the embedding of one micro-batch of the LM: 8 sequences of 2048 tokens
        dict(name="dropout_large", op="dropout", mode="train", type="bf16", N=8 * 2048 * 2048, p=0.1),
        # the LM's feed-forward for the eight sequences of a decoding step: every weight read once
        dict(name="ffn_decode", op="ffn", mode="serve", type="bf16", T=8, D=2048, F=8192, act="silu"),
        # the ViT's global batch: 512 images of 64 patches, short rows and a long sum over tokens
        dict(name="ffn_vit_train", op="ffn", mode="train", type="fp16", T=32768, D=384, F=1536, act="gelu_tanh"),
        # the LM's micro-batch: 8 sequences of 2048 tokens
        dict(name="ffn_lm_train", op="ffn", mode="train", type="bf16", T=16384, D=2048, F=8192, act="silu"),
        # ragged everywhere, float32
        dict(name="ffn_odd", op="ffn", mode="train", type="fp32", T=517, D=333, F=887, act="silu"),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _ragged(rng, lo, hi, grain):
    """As _spread; two times in three a multiple of `grain`, else any number."""
    v = _spread(rng, lo, hi)
    return v if rng.random() < 1 / 3 else max(grain, v // grain * grain)


def draw(rng):
    op = rng.choice(["read_norm", "write_norm", "dropout", "ffn"])
    case = dict(op=op, mode=rng.choice(["serve", "train"]), type=rng.choice(["bf16", "fp16", "fp32"]))
    if op == "dropout":
        case.update(N=_spread(rng, 1, 8 * 2048 * 2048), p=rng.choice([0.1, 0.5, round(rng.uniform(0.01, 0.9), 3)]))
        return case
    if op == "ffn":
        case.update(D=_ragged(rng, 64, 2048, 64), F=_ragged(rng, 64, 8192, 64), act=rng.choice(["silu", "gelu_tanh"]))
        # float32 products have no tensor cores to run on: fewer of them
        most = 2e10 if case["type"] == "fp32" else 16384 * 2048 * 8192
        case["T"] = _spread(rng, 1, max(1, min(32768, int(most / (case["D"] * case["F"])))))
        return case
    n = rng.randint(1, 8)
    case.update(n=n, m=rng.randint(1, min(n, 4)), D=_ragged(rng, 16, 4096, 64), norm=rng.choice(["rms", "layer"]),
                bias=rng.random() < 0.5)
    most = 16384 * 4 * 768 * (2 if case["type"] != "fp32" else 1)
    case["T"] = _spread(rng, 1, max(1, most // (case["n"] * case["D"])))
    if op == "write_norm":
        case.update(gate=rng.choice(["", "linear", "sigmoid"]), scale=rng.random() < 0.5, proj=rng.random() < 0.3,
                    p=rng.choice([0.0, 0.1, 0.3]))
    return case


# -------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    g = _generator(seed)
    dt = TYPES[case["type"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)

    s = dict(case=case, seed=int(seed) * 1000003 + 17, offset=5)
    if case["op"] == "dropout":
        s["x"], s["g"] = normal(case["N"], dtype=dt), normal(case["N"], dtype=dt)
    elif case["op"] == "ffn":
        T, D, F = case["T"], case["D"], case["F"]
        s["x"] = normal(T, D, dtype=dt)
        s["w_gate"] = normal(F, D, std=D ** -0.5, dtype=dt)
        s["w_up"] = normal(F, D, std=D ** -0.5, dtype=dt)
        s["w_down"] = normal(D, F, std=F ** -0.5, dtype=dt)
        s["g"] = normal(T, D, dtype=dt)
    else:
        T, n, m, D = (case[k] for k in ("T", "n", "m", "D"))
        # a residual stream whose tokens differ in size
        s["x"] = (normal(T, n, D) * torch.exp(normal(T, 1, 1, std=0.5))).to(dt)
        s["weight"] = normal(m * D, std=0.1, mean=1.0)
        s["bias"] = normal(m * D, std=0.1) if case["bias"] else None
        if case["op"] == "read_norm":
            s["R"] = torch.sigmoid(normal(T, m, n))
            s["g"] = normal(T, m, D, dtype=dt)
        else:
            # near the identity, as a layer's transition is
            s["H"] = torch.eye(n, device="cuda") + normal(T, n, n, std=0.2)
            s["W"] = 2 * torch.sigmoid(normal(T, n, m))
            s["f"] = (normal(T, m, D) * torch.exp(normal(T, 1, 1, std=0.5))).to(dt)
            s["gate"] = normal(T, m, D, dtype=dt) if case["gate"] else None
            s["scale"] = normal(m * D, std=0.02, mean=0.1) if case["scale"] else None
            v = normal(T, n)
            s["v"] = v / v.norm(dim=-1, keepdim=True) if case["proj"] else None
            s["g"] = normal(T, n, D, dtype=dt)
    return s


#: The inputs of each operator that have a gradient, in the order they are returned.
LEAVES = {
    "read_norm": ("R", "x", "weight", "bias"),
    "write_norm": ("H", "x", "W", "f", "v", "weight", "bias", "gate", "scale"),
    "dropout": ("x",),
    "ffn": ("x", "w_gate", "w_up", "w_down"),
}


# ---------------------------------------------------------------- plain form
def _philox(index, seed, offset):
    """Philox 4x32-10: the 32-bit word of each element (int64, 0 .. 2^32 - 1).
    Counter (element / 4, offset), key seed; element i takes word i mod 4."""
    low = 0xFFFFFFFF
    block = index >> 2
    c = [block & low, block >> 32, torch.full_like(block, offset & low), torch.full_like(block, (offset >> 32) & low)]
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57  # the low 64 bits, in two's complement
        c = [(b >> 32) & low ^ c[1] ^ k0, b & low, (a >> 32) & low ^ c[3] ^ k1, a & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    word = index & 3
    return torch.where(word < 2, torch.where(word == 0, c[0], c[1]), torch.where(word == 2, c[2], c[3]))


def _keep(shape, p, seed, offset, device):
    index = torch.arange(math.prod(shape), device=device)
    return (_philox(index, seed, offset) >= int(p * 2 ** 32)).view(shape)


def _normed(u, kind, eps=1e-6):
    if kind == "layer":
        u = u - u.mean(-1, keepdim=True)
    return u * (u.square().mean(-1, keepdim=True) + eps).rsqrt()


def _act(a, kind):
    if kind == "silu":
        return a / (1 + torch.exp(-a))
    return 0.5 * a * (1 + torch.tanh(math.sqrt(2 / math.pi) * (a + 0.044715 * a * a * a)))


def _plain(s, t):
    """The operator's output in 32 bits from its inputs `t` in 32 bits."""
    case = s["case"]
    if case["op"] == "dropout":
        kept = _keep(t["x"].shape, case["p"], s["seed"], s["offset"], t["x"].device)
        return torch.where(kept, t["x"] * (1 / (1 - case["p"])), 0.0)
    if case["op"] == "ffn":
        return (_act(t["x"] @ t["w_gate"].mT, case["act"]) * (t["x"] @ t["w_up"].mT)) @ t["w_down"].mT
    T, m, D = case["T"], case["m"], case["D"]
    u = t["R"] @ t["x"] if case["op"] == "read_norm" else t["f"]
    z = _normed(u.reshape(T, m * D), case["norm"]) * t["weight"]
    if t["bias"] is not None:
        z = z + t["bias"]
    if case["op"] == "read_norm":
        return z.view(T, m, D)
    if t["gate"] is not None:
        a = t["gate"].reshape(T, m * D)
        z = z * (1 / (1 + torch.exp(-a)) if case["gate"] == "sigmoid" else a)
    if t["scale"] is not None:
        z = z * t["scale"]
    if case["p"]:
        kept = _keep(z.shape, case["p"], s["seed"], s["offset"], z.device)
        z = torch.where(kept, z * (1 / (1 - case["p"])), 0.0)
    H = t["H"]
    if t["v"] is not None:
        v = t["v"].unsqueeze(-1)
        H = H + (v - H @ v) @ v.mT
    return H @ t["x"] + t["W"] @ z.view(T, m, D)


def _own(s, t):
    from hyperconnections_b200 import ops

    case = s["case"]
    if case["op"] == "dropout":
        return ops.hc_dropout(t["x"], case["p"], s["seed"], s["offset"])
    if case["op"] == "ffn":
        return ops.gated_ffn(t["x"], t["w_gate"], t["w_up"], t["w_down"], activation=case["act"])
    if case["op"] == "read_norm":
        return ops.hc_read_norm(t["R"], t["x"], t["weight"], t["bias"], norm=case["norm"], eps=1e-6)
    return ops.hc_mix_write_norm(t["H"], t["x"], t["W"], t["f"], t["v"], norm=case["norm"], weight=t["weight"],
                                 bias=t["bias"], eps=1e-6, gate=t["gate"], gate_activation=case["gate"] or "linear",
                                 scale=t["scale"], dropout_p=case["p"], seed=s["seed"], offset=s["offset"])


def run(s):
    case = s["case"]
    names = LEAVES[case["op"]]
    train = case["mode"] == "train"
    t = {k: None if s[k] is None else s[k].detach() for k in names}
    if not own:
        t = {k: None if a is None else a.float() for k, a in t.items()}
    if not train:
        with torch.no_grad():
            return [(_own if own else _plain)(s, t).to(s["x"].dtype)]
    t = {k: None if a is None else a.detach().requires_grad_() for k, a in t.items()}
    out = (_own if own else _plain)(s, t)
    has = [k for k in names if t[k] is not None]
    grads = torch.autograd.grad(out, [t[k] for k in has], s["g"] if own else s["g"].float())
    return [out.detach().to(s["x"].dtype)] + [a.to(s[k].dtype) for k, a in zip(has, grads)]


# ---------------------------------------------------------------------- work
def work(case):
    es = 4 if case["type"] == "fp32" else 2
    train = case["mode"] == "train"
    if case["op"] == "dropout":
        N = case["N"]
        return {"bytes": (4 if train else 2) * es * N, "flops": (2 if train else 1) * N}
    if case["op"] == "ffn":
        T, D, F = case["T"], case["D"], case["F"]
        moved = 2 * T * D + 3 * D * F + ((2 * T * D + 3 * D * F) if train else 0)
        return {"bytes": es * moved, "flops": (18 if train else 6) * T * D * F}
    T, n, m, D = (case[k] for k in ("T", "n", "m", "D"))
    E = m * D
    if case["op"] == "read_norm":
        params = E * (1 + case["bias"])
        stream, small = T * D * (n + m), T * m * n + params  # x in, y out; R and the norm's parameters in
        flops = T * D * (2 * m * n + 8 * m)
        if train:
            stream, small, flops = 2 * stream, 2 * small, flops + T * D * (6 * m * n + 12 * m)
        return {"bytes": es * stream + 4 * small, "flops": flops}
    gate = 1 if case["gate"] else 0
    params = E * (1 + case["bias"] + case["scale"])
    stream = T * D * (2 * n + m + m * gate)
    small = T * (n * n + n * m + (n if case["proj"] else 0)) + params
    flops = T * D * (2 * n * n + 2 * n * m + 8 * m)
    if train:
        stream, small, flops = 2 * stream, 2 * small, flops + T * D * (4 * n * n + 6 * n * m + 16 * m)
    return {"bytes": es * stream + 4 * small, "flops": flops}


# --------------------------------------------------------------------- exact
def _words(count, seed, offset):
    """Philox 4x32-10 by its definition, a block of four words at a time."""
    mask = 0xFFFFFFFF
    blocks = torch.arange((count + 3) // 4, device="cuda", dtype=torch.int64)
    x0, x1 = blocks.bitwise_and(mask), blocks.bitwise_right_shift(32)
    x2, x3 = torch.full_like(blocks, offset % 2 ** 32), torch.full_like(blocks, offset // 2 ** 32 % 2 ** 32)

    def product(a, b):  # (high, low) of 32 x 32 bits by 16-bit halves, so that nothing wraps
        al, ah, bl, bh = a & 0xFFFF, a >> 16, b & 0xFFFF, b >> 16
        mid = al * bh + ((al * bl) >> 16)
        mid2 = ah * bl + (mid & 0xFFFF)
        return ah * bh + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xFFFF) << 16) | ((al * bl) & 0xFFFF)

    for i in range(10):
        h0, l0 = product(x0, 0xD2511F53)
        h2, l2 = product(x2, 0xCD9E8D57)
        k0, k1 = (seed + i * 0x9E3779B9) % 2 ** 32, (seed // 2 ** 32 + i * 0xBB67AE85) % 2 ** 32
        x0, x1, x2, x3 = h2 ^ x1 ^ k0, l2, h0 ^ x3 ^ k1, l0
    return torch.stack([x0, x1, x2, x3], 1).reshape(-1)[:count]


def _factor(count, p, seed, offset):
    """What dropout multiplies each value with: 0 or 1 / (1 - p)."""
    if not p:
        return 1.0
    return (_words(count, seed, offset) >= math.floor(p * 2 ** 32)).double() / (1 - p)


def _exact_norm(u, weight, bias, kind, eps=1e-6):
    mean = u.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(u[:, :1])
    rstd = ((u - mean).pow(2).mean(1, keepdim=True) + eps).pow(-0.5)
    xhat = (u - mean) * rstd
    return xhat, rstd, xhat * weight + (0 if bias is None else bias)


def _exact_norm_back(q, xhat, rstd, kind):
    """The gradient before the norm from the gradient q of xhat."""
    d = q - xhat * (q * xhat).mean(1, keepdim=True)
    if kind == "layer":
        d = d - q.mean(1, keepdim=True)
    return d * rstd


def _exact_ffn(case, x, wg, wu, wd, g):
    a, b = x @ wg.T, x @ wu.T
    if case["act"] == "silu":
        sig = torch.sigmoid(a)
        act, der = a * sig, sig * (1 + a * (1 - sig))
    else:
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (a + 0.044715 * a ** 3))
        act, der = 0.5 * a * (1 + th), 0.5 * (1 + th) + 0.5 * a * (1 - th ** 2) * c * (1 + 3 * 0.044715 * a ** 2)
    h = act * b
    out = [h @ wd.T]
    if case["mode"] == "train":
        dh = g @ wd
        da, db = dh * b * der, dh * act
        out += [da @ wg + db @ wu, da.T @ x, db.T @ x, g.T @ h]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: a.double() for k, a in s.items() if torch.is_tensor(a)}
    g, train = d["g"], case["mode"] == "train"
    if case["op"] == "dropout":
        factor = _factor(case["N"], case["p"], s["seed"], s["offset"])
        return [d["x"] * factor] + ([g * factor] if train else [])
    if case["op"] == "ffn":
        return _exact_ffn(case, d["x"], d["w_gate"], d["w_up"], d["w_down"], g)
    T, m, D = case["T"], case["m"], case["D"]
    bias, weight, x = d.get("bias"), d["weight"], d["x"]
    if case["op"] == "read_norm":
        u = torch.einsum("tkj,tjd->tkd", d["R"], x).reshape(T, m * D)
        xhat, rstd, y = _exact_norm(u, weight, bias, case["norm"])
        out = [y.view(T, m, D)]
        if train:
            gf = g.reshape(T, m * D)
            du = _exact_norm_back(gf * weight, xhat, rstd, case["norm"]).view(T, m, D)
            out += [torch.einsum("tkd,tjd->tkj", du, x), torch.einsum("tkj,tkd->tjd", d["R"], du), (gf * xhat).sum(0)]
            out += [gf.sum(0)] if bias is not None else []
        return out
    H, W, v = d["H"], d["W"], d.get("v")
    xhat, rstd, b = _exact_norm(d["f"].reshape(T, m * D), weight, bias, case["norm"])
    a = da = torch.ones_like(b)
    if case["gate"]:
        a = d["gate"].reshape(T, m * D)
        if case["gate"] == "sigmoid":
            a = torch.sigmoid(a)
            da = a * (1 - a)
    scale = d.get("scale", torch.ones_like(weight))
    drop = _factor(b.numel(), case["p"], s["seed"], s["offset"])
    drop = drop.view_as(b) if torch.is_tensor(drop) else torch.full_like(b, drop)
    z = (scale * a * b * drop).view(T, m, D)
    out_x = torch.einsum("tij,tjd->tid", H, x) + torch.einsum("tik,tkd->tid", W, z)
    if v is not None:
        c = v - torch.einsum("tij,tj->ti", H, v)
        vx = torch.einsum("tj,tjd->td", v, x)
        out_x = out_x + torch.einsum("ti,td->tid", c, vx)
    out = [out_x]
    if not train:
        return out
    gH = torch.einsum("tid,tjd->tij", g, x)
    gx = torch.einsum("tij,tid->tjd", H, g)
    gv = None
    if v is not None:
        cg = torch.einsum("ti,tid->td", c, g)
        gx = gx + torch.einsum("tj,td->tjd", v, cg)
        gc = torch.einsum("tid,td->ti", g, vx)
        gv = gc - torch.einsum("tij,ti->tj", H, gc) + torch.einsum("td,tjd->tj", cg, x)
        gH = gH - torch.einsum("ti,tj->tij", gc, v)
    gz = (torch.einsum("tik,tid->tkd", W, g).reshape(T, m * D)) * drop
    inner = gz * a
    out += [gH, gx, torch.einsum("tid,tkd->tik", g, z),
            _exact_norm_back(inner * scale * weight, xhat, rstd, case["norm"]).view(T, m, D)]
    out += [gv] if v is not None else []
    out += [(inner * scale * xhat).sum(0)]
    out += [(inner * scale).sum(0)] if bias is not None else []
    out += [(gz * scale * b * da).view(T, m, D)] if case["gate"] else []
    out += [(inner * b).sum(0)] if "scale" in d else []
    return out
