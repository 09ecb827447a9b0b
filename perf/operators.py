"""Measured cases of the transformer-block operators: layer norm, rotary positions over several axes, and the linear
layer with its fused epilogue -- each with its backward pass.

Every case is one pass through one operator of `diffusionmodel_amd.ops`.  `run` computes it either in its plain form
(elementary torch operations in 32 bits, angles in 64) or, with `own` set, through the library's kernels; `exact`
states the same in 64 bits, written apart.
"""
import math

import torch

own = False

_ops = None


def _own_ops():
    global _ops
    if _ops is None:
        from diffusionmodel_amd import ops
        _ops = ops
    return _ops


# ---- cases ------------------------------------------------------------------------------------------------------------
def _ln(name, rows, C, dtype, **kw):
    c = {"name": name, "op": "ln_fwd", "rows": rows, "C": C, "dtype": dtype, "stats": False}
    c.update(kw)
    return c


def _rope(name, B, grid, Hq, Hk, D, dtype, **kw):
    c = {"name": name, "op": "rope", "B": B, "T": grid[0], "Y": grid[1], "X": grid[2], "Hq": Hq, "Hk": Hk, "D": D,
         "dtype": dtype, "layout": "half", "inverse": False, "offset": 0, "rotated": D}
    c.update(kw)
    return c


def _lin(name, M, K, N, dtype, **kw):
    c = {"name": name, "op": "linear", "M": M, "K": K, "N": N, "dtype": dtype, "act": "none", "res": False,
         "save_pre": False, "order": "kn"}
    c.update(kw)
    return c


def listed():
    return [
        # the norm of four images' time vectors: nothing but latency
        _ln("ln_time_vectors", 4, 256, "fp32"),
        # tokens of the bottleneck level (64 images of 16x16 pixels, 256 channels) in a training step
        _ln("ln_tokens_train", 16384, 256, "bf16", stats=True),
        # odd sizes: rows that are not 16-byte aligned, a prime number of them
        _ln("ln_odd_f32", 20011, 1031, "fp32", stats=True),
        # backward pass of a wide pre-norm block, the residual branch's gradient added on the way
        _ln("ln_bwd_wide", 65536, 1024, "bf16", op="ln_bwd", add=True),
        # the reference's own latents leave ONE token per image at the bottleneck
        _rope("rope_one_token", 4, (1, 1, 1), 4, 4, 64, "bf16"),
        # image tokens, q and k as slices of the fused projection
        _rope("rope_images", 64, (1, 16, 16), 4, 4, 64, "bf16"),
        # gradients of a video's queries and shared keys: time, height and width, adjacent pairs
        _rope("rope_video_bwd", 2, (8, 32, 32), 16, 4, 128, "fp32", layout="interleaved", inverse=True),
        # the time MLP's first layer for a batch of four: one pass over the weights
        _lin("linear_time", 4, 256, 2048, "bf16", act="relu"),
        # expansion of the bottleneck's tokens in a training step, pre-activation kept
        _lin("linear_tokens_train", 16384, 256, 1024, "bf16", act="gelu", save_pre=True),
        # projection back onto the residual stream, many tokens
        _lin("linear_wide_res", 65536, 4096, 1024, "bf16", res=True),
        # both products and the activation of an expansion's backward pass
        _lin("linear_bwd_wide", 16384, 1024, 4096, "bf16", op="linear_bwd", act="gelu"),
        # f32 with sizes that no tile divides
        _lin("linear_bwd_odd_f32", 1001, 321, 643, "fp32", op="linear_bwd", act="silu"),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A size over [lo, hi]: as it falls, or a multiple of 8 or 64 as layer widths mostly are."""
    v = _logint(rng, lo, hi)
    m = rng.choice((1, 8, 64))
    return max(m, v // m * m) if m <= hi else v


def draw(rng):
    op = rng.choice(("ln_fwd", "ln_bwd", "rope", "linear", "linear_bwd"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    if op in ("ln_fwd", "ln_bwd"):
        C = _size(rng, 8, 8192)
        rows = _logint(rng, 1, min(200000, (1 << 26) // C))
        c = _ln("", rows, C, dtype, op=op)
        if op == "ln_fwd":
            c["stats"] = rng.random() < 0.5
        else:
            c["add"] = rng.random() < 0.5
    elif op == "rope":
        D = rng.choice((32, 40, 64, 72, 96, 128, 256))
        Hk = rng.choice((1, 2, 4, 8))
        Hq = Hk * rng.choice((1, 1, 2, 4))
        T = rng.randint(1, 16) if rng.random() < 0.4 else 1
        Y, X = _logint(rng, 1, 48), _logint(rng, 1, 48)
        B = max(1, min(_logint(rng, 1, 64), (1 << 25) // (T * Y * X * (Hq + 2 * Hk) * D)))
        c = _rope("", B, (T, Y, X), Hq, Hk, D, dtype, layout=rng.choice(("half", "interleaved")),
                  inverse=rng.random() < 0.4, offset=rng.choice((0, 0, 1000, 1000000)),
                  rotated=rng.choice((D, D, D // 2 // 2 * 2)))
    else:
        K = _size(rng, 16, 4096)
        N = _size(rng, 16, 4096)
        M = _logint(rng, 1, max(1, min(65536, int(1.2e11 / (2.0 * K * N) / (2 if op == "linear_bwd" else 1)
                                                 / (4 if dtype == "fp32" else 1)))))
        c = _lin("", M, K, N, dtype, op=op, act=rng.choice(("none", "silu", "relu", "gelu")),
                 order=rng.choice(("kn", "kn", "nk")))
        if op == "linear":
            c["res"] = rng.random() < 0.4
            c["save_pre"] = rng.random() < 0.4
    del c["name"]
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _dt(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _sections(case):
    """Rotated pairs of each axis: a quarter for time and the rest shared by height and width, as far as it divides."""
    pairs = case["rotated"] // 2
    if case["T"] == 1:
        return (pairs - pairs // 2, pairs // 2)
    yx = pairs * 3 // 8
    return (pairs - 2 * yx, yx, yx)


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _dt(case)

    def rn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    op = case["op"]
    st = {"case": case}
    if op in ("ln_fwd", "ln_bwd"):
        R, C = case["rows"], case["C"]
        # per-channel scales and offsets as a trained stream has them: a few loud channels, none centred
        scale = torch.exp(0.5 * rn(C))
        x = rn(R, C).mul_(scale).add_(rn(C)).to(dt)
        st.update(x=x, w=1.0 + 0.1 * rn(C), b=0.1 * rn(C), eps=1e-5)
        if op == "ln_bwd":
            xf = x.float()
            mean = xf.mean(1)
            st.update(dy=rn(R, C).to(dt), mean=mean, add=rn(R, C).to(dt) if case["add"] else None,
                      rstd=torch.rsqrt((xf - mean[:, None]).square().mean(1) + st["eps"]))
    elif op == "rope":
        B, N, D = case["B"], case["T"] * case["Y"] * case["X"], case["D"]
        Hq, Hk = case["Hq"], case["Hk"]
        qkv = rn(B, N, Hq + 2 * Hk, D).to(dt)
        sec = _sections(case)
        t, y, x = torch.meshgrid(torch.arange(case["T"]), torch.arange(case["Y"]), torch.arange(case["X"]), indexing="ij")
        axes = [t, y, x] if len(sec) == 3 else [y, x]
        pos = torch.stack([a.reshape(-1) for a in axes]).to(torch.int32) + case["offset"]
        inv = torch.cat([torch.tensor([10000.0 ** (-j / n) for j in range(n)], dtype=torch.float32) for n in sec])
        axis = torch.tensor([a for a, n in enumerate(sec) for _ in range(n)])
        st.update(qkv=qkv, q=qkv[:, :, :Hq], k=qkv[:, :, Hq:Hq + Hk], pos=pos.to(dev), inv=inv.to(dev), axis=axis.to(dev),
                  sections=sec)
    else:
        M, K, N = case["M"], case["K"], case["N"]
        w = (rn(K, N) * K ** -0.5).to(dt)
        if case["order"] == "nk":
            w = w.t().contiguous().t()          # [K, N] whose memory holds [N, K]
        st.update(x=rn(M, K).to(dt), w=w, b=0.1 * rn(N))
        if op == "linear":
            st["res"] = rn(M, N).to(dt) if case["res"] else None
        else:
            st.update(dy=rn(M, N).to(dt), pre=rn(M, N).to(dt) if case["act"] != "none" else None)
    return st


# ---- plain forms ------------------------------------------------------------------------------------------------------
def _plain_ln(x, w, b, eps):
    xf = x.float()
    mean = xf.mean(1, keepdim=True)
    xc = xf - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(1, keepdim=True) + eps)
    return (xc * rstd * w + b).to(x.dtype), mean[:, 0], rstd[:, 0]


def _plain_ln_bwd(dy, x, mean, rstd, w, add):
    d = dy.float()
    xh = (x.float() - mean[:, None]) * rstd[:, None]
    gw = d * w
    dx = rstd[:, None] * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
    if add is not None:
        dx = dx + add.float()
    return dx.to(x.dtype), (d * xh).sum(0), d.sum(0)


def _plain_rotate(x, cos, sin, pairs, layout):
    xf = x.float()
    rot, rest = xf[..., :2 * pairs], xf[..., 2 * pairs:]
    if layout == "half":
        a, b = rot[..., :pairs], rot[..., pairs:]
        out = torch.cat([a * cos - b * sin, a * sin + b * cos, rest], -1)
    else:
        a, b = rot[..., 0::2], rot[..., 1::2]
        out = torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), rest], -1)
    return out.to(x.dtype)


def _plain_act(z, act):
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "relu":
        return torch.clamp(z, min=0.0)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z


def _plain_dact(z, act):
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    if act == "relu":
        return (z > 0).to(z.dtype)
    return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5


def run(state):
    c = state["case"]
    return _run_own(c, state) if own else _run_plain(c, state)


def _run_plain(c, s):
    op = c["op"]
    if op == "ln_fwd":
        y, mean, rstd = _plain_ln(s["x"], s["w"], s["b"], s["eps"])
        return (y, mean, rstd) if c["stats"] else y
    if op == "ln_bwd":
        return _plain_ln_bwd(s["dy"], s["x"], s["mean"], s["rstd"], s["w"], s["add"])
    if op == "rope":
        ang = s["pos"].double()[s["axis"]].t() * s["inv"].double()     # [N, pairs]
        cos, sin = torch.cos(ang).float()[None, :, None], torch.sin(ang).float()[None, :, None]
        if c["inverse"]:
            sin = -sin
        p = s["inv"].numel()
        return _plain_rotate(s["q"], cos, sin, p, c["layout"]), _plain_rotate(s["k"], cos, sin, p, c["layout"])
    if op == "linear":
        z = s["x"].float() @ s["w"].float() + s["b"]
        if s["res"] is not None:
            z = z + s["res"].float()
        out = _plain_act(z, c["act"]).to(_dt(c))
        return (out, z.to(_dt(c))) if c["save_pre"] else out
    dz = s["dy"].float()
    if c["act"] != "none":
        dz = dz * _plain_dact(s["pre"].float(), c["act"])
    return ((dz @ s["w"].float().t()).to(_dt(c)), (s["x"].float().t() @ dz).to(_dt(c)), dz.sum(0))


# ---- the library's calls ----------------------------------------------------------------------------------------------
def _run_own(c, s):
    ops = _own_ops()
    op = c["op"]
    if op == "ln_fwd":
        return ops.layer_norm(s["x"], s["w"], s["b"], eps=s["eps"], stats=c["stats"])
    if op == "ln_bwd":
        return ops.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["w"], add=s["add"])
    if op == "rope":
        return ops.rope(s["q"], s["k"], s["pos"], s["inv"], sections=s["sections"], layout=c["layout"],
                        inverse=c["inverse"])
    if op == "linear":
        return ops.linear(s["x"], s["w"], s["b"], act=c["act"], res=s["res"], save_pre=c["save_pre"])
    dx, dw, db, _ = ops.linear_backward(s["dy"], s["x"], s["w"], pre=s["pre"], act=c["act"])
    return dx, dw, db


# ---- work -------------------------------------------------------------------------------------------------------------
def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    op = case["op"]
    if op == "ln_fwd":
        n = case["rows"] * case["C"]
        return {"bytes": 2 * n * es + 8 * case["C"] + (8 * case["rows"] if case["stats"] else 0), "flops": 8 * n}
    if op == "ln_bwd":
        n = case["rows"] * case["C"]
        return {"bytes": (4 if case["add"] else 3) * n * es + 12 * case["C"] + 8 * case["rows"], "flops": 14 * n}
    if op == "rope":
        N = case["T"] * case["Y"] * case["X"]
        n = case["B"] * N * (case["Hq"] + case["Hk"]) * case["D"]
        return {"bytes": 2 * n * es + 4 * N * len(_sections(case)) + 2 * case["rotated"], "flops": 3 * n}
    M, K, N = case["M"], case["K"], case["N"]
    if op == "linear":
        return {"bytes": (M * K + K * N + M * N * (1 + case["res"] + case["save_pre"])) * es + 4 * N,
                "flops": 2 * M * K * N}
    return {"bytes": (2 * M * K + 2 * K * N + M * N * (2 if case["act"] != "none" else 1)) * es + 4 * N,
            "flops": 4 * M * K * N}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "ln_fwd":
        x = s["x"].double()
        var, mean = torch.var_mean(x, dim=-1, correction=0)
        r = (var + s["eps"]).pow(-0.5)
        y = torch.addcmul(s["b"].double(), (x - mean.unsqueeze(-1)) * r.unsqueeze(-1), s["w"].double())
        return (y, mean, r) if case["stats"] else y
    if op == "ln_bwd":
        # y = xh w + b with xh = (x - m) r: dx is r times the part of g = dy w orthogonal to 1 and to xh
        x, dy = s["x"].double(), s["dy"].double()
        r = s["rstd"].double().unsqueeze(-1)
        xh = (x - s["mean"].double().unsqueeze(-1)) * r
        g = dy * s["w"].double()
        C = case["C"]
        s1 = g.sum(-1, keepdim=True) / C
        s2 = torch.linalg.vecdot(g, xh).unsqueeze(-1) / C
        dx = (g - s1 - s2 * xh) * r
        if s["add"] is not None:
            dx = dx + s["add"].double()
        return dx, torch.einsum("rc,rc->c", dy, xh), dy.sum(0)
    if op == "rope":
        # a rotation of the plane (a, b) by the angle t is a complex product with e^(i t)
        sec = s["sections"]
        parts, j = [], 0
        for ax, n in enumerate(sec):
            parts.append(torch.outer(s["pos"][ax].double(), s["inv"][j:j + n].double()))
            j += n
        ang = torch.cat(parts, 1)
        e = torch.polar(torch.ones_like(ang), -ang if case["inverse"] else ang)[:, None, :]
        P = case["rotated"] // 2

        def turn(x):
            x = x.double().clone()
            v = x[..., :2 * P]
            if case["layout"] == "half":
                z = torch.complex(v[..., :P].contiguous(), v[..., P:].contiguous()) * e
                x[..., :P], x[..., P:2 * P] = z.real, z.imag
            else:
                z = torch.view_as_complex(v.reshape(*v.shape[:-1], P, 2).contiguous()) * e
                x[..., :2 * P] = torch.view_as_real(z).flatten(-2)
            return x
        return turn(s["q"]), turn(s["k"])
    x, w = s["x"].double(), s["w"].double()
    act = case["act"]
    if op == "linear":
        z = torch.addmm(s["b"].double(), x, w)
        if s["res"] is not None:
            z += s["res"].double()
        out = {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu,
               "gelu": torch.nn.functional.gelu}[act](z)
        return (out, z) if case["save_pre"] else out
    dz = s["dy"].double()
    if act != "none":
        p = s["pre"].double()
        if act == "relu":
            dz = torch.where(p > 0, dz, 0.0)
        elif act == "silu":
            sg = torch.sigmoid(p)
            dz = dz * torch.addcmul(sg, p, sg * torch.sigmoid(-p))
        else:
            dz = dz * (0.5 * torch.erfc(-p / math.sqrt(2.0)) + p * torch.exp(-p * p / 2) / math.sqrt(2.0 * math.pi))
    return dz @ w.t(), x.t() @ dz, dz.sum(0)
