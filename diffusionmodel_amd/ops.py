"""Kernel-level operators of libldm_hip.so on device tensors (include/ldm_hip.h).

ConvOp, batchnorm_act: one convolution / batch norm of the UNet on NHWC tensors in the library's own layout.
layer_norm, rope, linear, each with its backward pass: what a transformer block over latent tokens needs around its
attention."""
from __future__ import annotations

import ctypes as C
import functools
import operator
import struct
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib

KINDS = {"conv3x3": 0, "conv3x3_s2": 1, "convT4x4_s2": 2, "conv1x1": 3}
ACTS = {None: 0, "none": 0, "silu": 1, "relu": 2}


def to_nhwc(x: torch.Tensor, dtype: str) -> torch.Tensor:
    """NCHW f32 -> contiguous NHWC tensor of the operator's element type."""
    td = torch.bfloat16 if dtype == "bf16" else torch.float32
    return x.permute(0, 2, 3, 1).contiguous().to(td)


def from_nhwc(y: torch.Tensor) -> torch.Tensor:
    return y.float().permute(0, 3, 1, 2).contiguous()


class ConvOp:
    """kind: 'conv3x3' | 'conv3x3_s2' | 'convT4x4_s2' | 'conv1x1'; weight in burn's layout for the kind
    ([Cout,Cin,3,3] | [Cin,Cout,4,4] | [Cout,Cin0+Cin1(,1,1)]); channel counts multiples of 64."""

    def __init__(self, kind: str, weight: torch.Tensor, bias: torch.Tensor, dtype: str = "bf16", cin1: int = 0):
        self._lib = _lib.load()
        self.kind, self.dtype = kind, dtype
        self.code = _lib.LDM_BF16 if dtype == "bf16" else _lib.LDM_F32
        w = weight.detach().to("cpu", torch.float32).contiguous()
        b = bias.detach().to("cpu", torch.float32).contiguous()
        if kind == "convT4x4_s2":
            cin, self.cout = w.shape[0], w.shape[1]
        else:
            self.cout, cin = w.shape[0], w.shape[1]
        self.cin0, self.cin1 = cin - cin1, cin1
        self._h = C.c_void_p()
        _lib.check(self._lib.ldm_conv_create(C.byref(self._h), KINDS[kind], self.code, self.cin0, self.cin1, self.cout,
                                             C.c_void_p(w.data_ptr()), C.c_void_p(b.data_ptr())))

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h:
            try:
                self._lib.ldm_conv_destroy(h)
            except Exception:
                pass

    def out_hw(self, H: int, W: int):
        if self.kind == "conv3x3_s2":
            return (H - 1) // 2 + 1, (W - 1) // 2 + 1
        if self.kind == "convT4x4_s2":
            return 2 * H, 2 * W
        return H, W

    def forward(self, x0: torch.Tensor, x1: Optional[torch.Tensor] = None, res: Optional[torch.Tensor] = None,
                act: Optional[str] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x0 [B,H,W,cin0], x1 [B,H,W,cin1] or None, res [B,Ho,Wo,cout] or None: contiguous NHWC device tensors."""
        td = torch.bfloat16 if self.dtype == "bf16" else torch.float32
        for t, c in ((x0, self.cin0), (x1, self.cin1)):
            if t is None:
                continue
            if not (t.is_cuda and t.is_contiguous() and t.dtype == td and t.dim() == 4 and t.shape[3] == c):
                raise ValueError("inputs must be contiguous NHWC device tensors of the operator's dtype and channels")
        if (x1 is None) != (self.cin1 == 0):
            raise ValueError("second source does not match the operator")
        B, H, W, _ = x0.shape
        Ho, Wo = self.out_hw(H, W)
        if out is None:
            out = torch.empty((B, Ho, Wo, self.cout), dtype=td, device=x0.device)
        if res is not None and not (res.is_contiguous() and res.dtype == td and tuple(res.shape) == tuple(out.shape)):
            raise ValueError("residual must match the output")
        stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
        p = lambda t: C.c_void_p(0 if t is None else t.data_ptr())  # noqa: E731
        _lib.check(self._lib.ldm_conv_forward(self._h, p(x0), p(x1), p(res), p(out), B, H, W, ACTS[act], stream))
        return out

    __call__ = forward


def batchnorm_act(h: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, act: Optional[str] = None,
                  res: Optional[torch.Tensor] = None, tvec: Optional[torch.Tensor] = None, eps: float = 1e-5,
                  dropout_p: float = 0.0, seed: int = 0, out: Optional[torch.Tensor] = None, stats_only: bool = False):
    """Training-mode BatchNorm + the ResidualBlock's tail on a contiguous NHWC device tensor h [B,H,W,C] (bf16 or
    f32): out = dropout(act(((h - mean) / sqrt(var + eps)) * gamma + beta + res) + tvec[b]) with the batch
    statistics of h (ldm_batchnorm_act; burn's BatchNorm on the autodiff backend, src/main.rs:374, 385, 1318).
    Returns (out, mean, var); out is None with stats_only."""
    if not (h.is_cuda and h.is_contiguous() and h.dim() == 4 and h.dtype in (torch.bfloat16, torch.float32)):
        raise ValueError("h must be a contiguous NHWC device tensor, bf16 or f32")
    B, H, W, Cc = h.shape
    code = _lib.LDM_BF16 if h.dtype == torch.bfloat16 else _lib.LDM_F32
    lib = _lib.load()
    g = gamma.detach().to(h.device, torch.float32).contiguous()
    b = beta.detach().to(h.device, torch.float32).contiguous()
    if g.numel() != Cc or b.numel() != Cc:
        raise ValueError("gamma and beta must hold one value per channel")
    nws = lib.ldm_batchnorm_ws_floats(code, B * H * W, Cc)
    if nws <= 0:
        raise ValueError("channel count not served")
    ws = torch.empty(nws, dtype=torch.float32, device=h.device)
    mean = torch.empty(Cc, dtype=torch.float32, device=h.device)
    var = torch.empty(Cc, dtype=torch.float32, device=h.device)
    if res is not None and not (res.is_contiguous() and res.dtype == h.dtype and tuple(res.shape) == tuple(h.shape)):
        raise ValueError("res must match h")
    if tvec is not None:
        tvec = tvec.detach().to(h.device, torch.float32).contiguous()
        if tuple(tvec.shape) != (B, Cc):
            raise ValueError("tvec must be [B, C]")
    if not stats_only and out is None:
        out = torch.empty_like(h)
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    p = lambda t: C.c_void_p(0 if t is None else t.data_ptr())  # noqa: E731
    _lib.check(lib.ldm_batchnorm_act(code, p(h), p(res), p(None if stats_only else out), B, H * W, Cc, p(g), p(b), eps,
                                     ACTS[act], p(tvec), dropout_p, seed & (2 ** 64 - 1), p(ws), p(mean), p(var), stream))
    return (None if stats_only else out), mean, var


# ---- operators of transformer blocks ---------------------------------------------------------------------------------
# Explicit forward and backward calls on tensors of one device, on that device's current stream; like every operator here
# they record no autograd graph, so a tensor that requires a gradient is refused while gradients are recorded.  Workspaces
# come from torch's allocator for the one call, so calls on several streams and captured graphs do not share them.
_TD = {torch.bfloat16: _lib.LDM_BF16, torch.float32: _lib.LDM_F32}
_F32 = (torch.float32,)
_REAL = (torch.float32, torch.bfloat16, torch.float16, torch.float64)
LINEAR_ACTS = {None: 0, "none": 0, "silu": 1, "relu": 2, "gelu": 3}
ROPE_LAYOUTS = {"half": 0, "interleaved": 1}
_POS_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}

# torch.cuda.current_stream() builds a Stream object (2.6 us, as much as a launch); the raw handle is what is needed.  Small
# calls are bound by what happens here before the launch, so the checks below take the ordinary case first.
_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _data(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _check_bits(name: str, t: torch.Tensor) -> None:
    """The library reads a tensor's memory: what torch keeps beside it would be lost without a word."""
    if t.is_neg():
        raise ValueError(f"{name} is a negated view whose memory holds the opposite values: call resolve_neg() on it first")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} carries a forward-mode tangent, which this operator does not propagate: unpack it first")


def _check(name: str, t, dev: int = -1, dtypes=_TD) -> int:
    """A device tensor of one of `dtypes`, on device `dev` (-1: any), that needs no gradient.  Returns its device."""
    if isinstance(t, torch.Tensor) and t.dtype in dtypes and not t.requires_grad and not t.is_neg() \
            and forward_ad._current_level < 0:
        d = t.get_device()
        if d >= 0 and (dev < 0 or d == dev):
            return d
    if isinstance(t, torch.Tensor):
        _check_bits(name, t)
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} is {t.dtype}, expected one of {tuple(str(d) for d in dtypes)}")
    if dev >= 0 and t.get_device() != dev:
        raise ValueError(f"{name} is on device {t.get_device()}, expected {dev}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which this operator does not record: call it under "
                         "torch.no_grad() and use the operator's backward function")
    return t.get_device()


def _rows(name: str, t: torch.Tensor) -> Tuple[int, int]:
    """(rows, row stride) of t [..., C] as one matrix; its last axis must be contiguous."""
    if t.is_contiguous():
        c = t.size(-1)
        return (t.numel() // c if c else 0), c
    if t.shape[-1] != 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous along its last axis")
    rows, stride = 1, None
    for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if n == 1:
            continue
        if stride is not None and s != stride * rows and rows > 0:
            raise ValueError(f"{name}: leading axes with strides {tuple(t.stride())} are not one run of rows; "
                             "make it contiguous")
        if stride is None:
            stride = s
        rows *= n
    return rows, (t.shape[-1] if stride is None else stride)


def _extent(t: torch.Tensor, dims) -> int:
    return 1 + sum((t.shape[d] - 1) * t.stride(d) for d in dims)


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether no element of a lies in b: their address ranges are apart, or, for two slices of one buffer, their blocks
    are apart within every step of the leading axes that they share."""
    if a.numel() == 0 or b.numel() == 0:
        return True
    if b.data_ptr() < a.data_ptr():
        a, b = b, a
    ea, eb = a.element_size(), b.element_size()
    gap = b.data_ptr() - a.data_ptr()
    if gap >= _extent(a, range(a.dim())) * ea:
        return True
    for lead in range(1, min(a.dim(), b.dim())):
        if a.shape[:lead] != b.shape[:lead] or a.stride()[:lead] != b.stride()[:lead] or ea != eb:
            return False
        room = gap + _extent(b, range(lead, b.dim())) * eb          # bytes of one step: both blocks side by side
        steps = sorted((s * ea, n) for s, n in zip(a.stride()[:lead], a.shape[:lead]) if n > 1)
        ok = gap >= _extent(a, range(lead, a.dim())) * ea
        for s, n in steps:
            ok = ok and s >= room
            room = s * n
        if ok:
            return True
    return False


def _check_out(name: str, out: torch.Tensor, shape, like: torch.Tensor, inputs, same: Optional[torch.Tensor] = None) -> None:
    """An output given by the caller: right shape and type, no element twice, apart from the inputs; `same` is an input
    that it may replace, as the very same view."""
    _check(name, out, like.get_device(), (like.dtype,))
    if tuple(out.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(out.shape)}, expected {tuple(shape)}")
    reach = 1
    for s, n in sorted((s, n) for n, s in zip(out.shape, out.stride()) if n > 1):
        if s < reach:
            raise ValueError(f"{name} holds elements more than once")
        reach = s * n
    if same is not None and not (same.data_ptr() == out.data_ptr() and same.stride() == out.stride()):
        inputs = tuple(inputs) + (same,)
    for t in inputs:
        if t is not None and not _apart(out, t):
            raise ValueError(f"{name} overlaps an input in memory")


def _params(name: str, t: Optional[torch.Tensor], n: int, dev: int) -> Optional[torch.Tensor]:
    """n contiguous f32 values on device `dev` (another floating type is converted), or None."""
    if t is None:
        return None
    _check(name, t, dev, _REAL)
    if t.dim() != 1 or t.numel() != n:
        raise ValueError(f"{name} must hold {n} values, has shape {tuple(t.shape)}")
    return t if t.dtype is torch.float32 and t.is_contiguous() else t.to(torch.float32).contiguous()


def _like(x: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of x's shape, type and device."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty_like(x, memory_format=torch.contiguous_format)


def _call(fn, dev: int, *args) -> None:
    """One library call on device `dev` and its current stream (the function's last argument)."""
    if dev == _device():
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc:
        _lib.check(rc)


def _columns(t: torch.Tensor) -> int:
    """Elements of t's last axis; the library's norms take up to 2^24 (and a larger count would not survive its 32 bits)."""
    if t.dim() < 1 or not 1 <= t.size(-1) <= 1 << 24:
        raise ValueError("x must have a last axis of 1 to 2^24 elements")
    return t.size(-1)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, out: Optional[torch.Tensor] = None, stats: bool = False):
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last axis of x [..., C] (bf16 or f32, last axis
    contiguous, leading axes one run of rows: ldm_layer_norm).  weight and bias hold C values and are used in f32.
    Returns y, or (y, mean, rstd) with `stats`: f32 of shape [...], what layer_norm_backward needs.
    `out` may be x itself."""
    dev = _check("x", x)
    shape = x.shape
    Cc = _columns(x)
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    rows, xs = _rows("x", x)
    w, b = _params("weight", weight, Cc, dev), _params("bias", bias, Cc, dev)
    if out is None:
        out, ys = _like(x), Cc
    else:
        _check_out("out", out, shape, x, (w, b), same=x)
        ys = _rows("out", out)[1]
    mean = rstd = None
    if stats:
        mean = x.new_empty(shape[:-1], dtype=torch.float32)
        rstd = torch.empty_like(mean)
    if rows:
        _call(_lib.load().ldm_layer_norm, dev, _TD[x.dtype], x.data_ptr(), xs, _data(w), _data(b), eps,
              out.data_ptr(), ys, _data(mean), _data(rstd), rows, Cc)
    return (out, mean, rstd) if stats else out


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: Optional[torch.Tensor] = None, add: Optional[torch.Tensor] = None,
                        param_grads: Optional[bool] = None):
    """Gradients of layer_norm (ldm_layer_norm_backward): (dx, dweight, dbias), dx in x's type, the parameters' in f32.
    mean and rstd are the forward pass's statistics; `add` (x's shape and type) is added to dx, the gradient that
    reaches x by the residual branch.  param_grads=False (the default without a weight) leaves dweight and dbias None."""
    dev = _check("x", x)
    Cc = _columns(x)
    for name, t in (("dy", dy), ("add", add)):
        if t is not None or name == "dy":
            _check(name, t, dev, (x.dtype,))
            if t.shape != x.shape:
                raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(x.shape)}")
    for name, t in (("mean", mean), ("rstd", rstd)):
        _check(name, t, dev, _F32)
        if t.shape != x.shape[:-1] or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous with shape {tuple(x.shape[:-1])}")
    rows, xs = _rows("x", x)
    dys = _rows("dy", dy)[1]
    adds = 0 if add is None else _rows("add", add)[1]
    w = _params("weight", weight, Cc, dev)
    if param_grads is None:
        param_grads = weight is not None
    dx = _like(x)
    lib = _lib.load()
    code = _TD[x.dtype]
    dw = db = ws = None
    if param_grads:
        dw = x.new_empty(Cc, dtype=torch.float32)
        db = torch.empty_like(dw)
        ws = x.new_empty(lib.ldm_layer_norm_ws_floats(code, rows, Cc), dtype=torch.float32)
    if rows or param_grads:
        _call(lib.ldm_layer_norm_backward, dev, code, dy.data_ptr(), dys, x.data_ptr(), xs, _data(add), adds,
              mean.data_ptr(), rstd.data_ptr(), _data(w), dx.data_ptr(), Cc, _data(dw), _data(db), _data(ws), rows, Cc)
    return dx, dw, db


def rope_frequencies(sections: Sequence[int], theta: float = 10000.0, shared: bool = False,
                     device: Optional[torch.device] = None) -> torch.Tensor:
    """Frequencies [sum(sections)] f32 for `rope`: each axis has a ladder of its own, theta^(-j / n) for pair j of its n
    pairs, or (shared) its section of one ladder over all pairs."""
    if len(sections) < 1 or any(int(n) != n or n < 0 for n in sections) or sum(sections) < 1:
        raise ValueError("sections must be non-negative pair counts, at least one pair in all")
    if not theta > 0.0:
        raise ValueError("theta must be positive")
    ladders = [sum(sections)] if shared else list(sections)
    f = torch.cat([theta ** (-torch.arange(n, dtype=torch.float64) / n) for n in ladders if n])
    return f.to(device=device, dtype=torch.float32)


def rope(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor,
         sections: Optional[Sequence[int]] = None, layout: str = "half", inverse: bool = False, out=None):
    """Rotary positions over one to four axes (ldm_rope).  q [B, N, Hq, D] and k [B, N, Hk, D] or None: bf16 or f32,
    any strides with D contiguous (slices of a fused projection need no copy).  positions [axes, N], or [B, axes, N]:
    int32, int64 or f32.  inv_freq [P] f32; sections: how many of the P pairs each axis turns (None: one axis turns all).
    layout "half" pairs (j, P + j), "interleaved" (2j, 2j + 1); elements behind 2P pass through.
    inverse=True turns back: applied to the gradients of the outputs it gives the gradients of q and k.
    Returns (q', k'), or q' if k is None; `out` = (q', k') or q' to write to, which may be the inputs themselves."""
    dev = _check("q", q)
    if k is not None:
        _check("k", k, dev, (q.dtype,))
    _check("inv_freq", inv_freq, dev, _F32)
    if inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous vector")
    _check("positions", positions, dev, _POS_TYPES)
    ok = None
    if out is None:
        oq = _like(q)
        if k is not None:
            ok = _like(k)
    else:
        oq, ok = (out, None) if k is None else out
        _check_out("out[0]", oq, q.shape, q, (k, positions, inv_freq), same=q)
        if k is not None:
            _check_out("out[1]", ok, k.shape, q, (q, oq, positions, inv_freq), same=k)
    if sections is not None:
        # (as whole numbers before the plans are searched, where 4.0 or a tensor would find what 4 left)
        try:
            sections = tuple(map(operator.index, sections))
        except TypeError:
            raise ValueError(f"sections must be whole numbers, got {sections}") from None
    strides, dims, pos_strides, sec, axes = _rope_plan(
        q.shape, q.stride(), None if k is None else k.shape, None if k is None else k.stride(), oq.stride(),
        None if k is None else ok.stride(), positions.shape, positions.stride(), inv_freq.numel(),
        sections, layout)
    if q.numel():
        _call(_lib.load().ldm_rope, dev, _TD[q.dtype], q.data_ptr(), _data(k), oq.data_ptr(), _data(ok), strides, *dims,
              positions.data_ptr(), _POS_TYPES[positions.dtype], pos_strides, inv_freq.data_ptr(), sec, axes,
              ROPE_LAYOUTS[layout], bool(inverse))
    return oq if k is None else (oq, ok)


@functools.lru_cache(maxsize=1024)
def _rope_plan(qs, sq, ks, sk, so, sok, ps, pp, P, sections, layout):
    """Checks the shapes and strides of a rope call and packs them for the library."""
    if len(qs) != 4:
        raise ValueError("q must be [B, N, heads, D]")
    B, N, Hq, D = qs
    Hk = 0
    if ks is None:
        sk = sok = (0, 0, 0, 1)
    else:
        if len(ks) != 4 or ks[0] != B or ks[1] != N or ks[3] != D:
            raise ValueError(f"k must be [{B}, {N}, heads, {D}], has shape {tuple(ks)}")
        Hk = ks[2]
    if max(B, N, Hq, Hk, D) >= 1 << 31:
        raise ValueError("B, N, heads and D must be below 2^31")
    if D < 1 or Hq < 1 or (ks is not None and Hk < 1) or (D > 1 and not sq[3] == sk[3] == so[3] == sok[3] == 1):
        raise ValueError("q, k and their outputs need at least one head and contiguous head vectors")
    sec = (P,) if sections is None else sections
    if not 1 <= len(sec) <= 4 or min(sec) < 0 or sum(sec) != P or P < 1 or 2 * P > D:
        raise ValueError(f"sections {sec} must hold one to four counts that add up to inv_freq's {P} pairs, at most D / 2")
    if len(ps) == 2:
        ps, pp = (B,) + tuple(ps), (0,) + tuple(pp)
    if len(ps) != 3 or ps[0] != B or ps[1] != len(sec) or ps[2] != N:
        raise ValueError(f"positions must be [{len(sec)}, {N}] or [{B}, {len(sec)}, {N}], has shape {tuple(ps)}")
    if layout not in ROPE_LAYOUTS:
        raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
    return (struct.pack("12l", *(tuple(sq[:3]) + tuple(sk[:3]) + tuple(so[:3]) + tuple(sok[:3]))), (B, N, Hq, Hk, D),
            struct.pack("3l", *pp), struct.pack(f"{len(sec)}i", *sec), len(sec))


def _weight_order(weight: torch.Tensor) -> Tuple[int, int]:
    """(order, leading stride) of a weight [K, N]: 0 for rows of N, 1 for a transposed weight (rows of K)."""
    K, N = weight.shape
    s0, s1 = weight.stride()
    if N == 1 or s1 == 1:
        return 0, (s0 if K > 1 else N)
    if K == 1 or s0 == 1:
        return 1, s1
    raise ValueError("weight must be contiguous along one of its axes")


def _check_linear(x: torch.Tensor, weight: torch.Tensor, act: Optional[str]) -> Tuple[int, int, int]:
    dev = _check("x", x)
    _check("weight", weight, dev, (x.dtype,))
    ws = weight.shape
    if len(ws) != 2 or min(ws) < 1:
        raise ValueError("weight must be [K, N] with K, N >= 1")
    if x.dim() < 1 or x.size(-1) != ws[0]:
        raise ValueError(f"x must be [..., {ws[0]}], has shape {tuple(x.shape)}")
    if act not in LINEAR_ACTS:
        raise ValueError(f"act must be one of {sorted(a for a in LINEAR_ACTS if a)}, got {act!r}")
    return dev, ws[0], ws[1]


@functools.lru_cache(maxsize=4096)
def _linear_ws(backward: bool, *shape: int) -> int:
    """Floats of workspace; shape = (type code, M, K, N, weight order)."""
    lib = _lib.load()
    return (lib.ldm_linear_backward_ws_floats if backward else lib.ldm_linear_ws_floats)(*shape)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, act: Optional[str] = None,
           res: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, save_pre: bool = False):
    """act(x @ weight + bias + res) (ldm_linear): x [..., K] and weight [K, N] (burn's Linear layout, or a transposed view
    of an [N, K] weight) in bf16 or f32, bias N values used in f32, res [..., N] in x's type, added before the activation
    like a convolution's; act None, 'silu', 'relu' or 'gelu' (z Phi(z), not the tanh form).  Products accumulate in f32.
    Activations before the last rounding: within 9 half steps of f32 of their value; in bf16 within 2^-11 (GELU: down to z = -9).
    Returns the output in x's type, or (output, z) with save_pre: z, the value before the activation, is what
    linear_backward needs with one.  `out` may be res itself.  Rows of a matrix may lie up to 2^21 elements apart."""
    dev, K, N = _check_linear(x, weight, act)
    M, ldx = _rows("x", x)
    order, ldw = _weight_order(weight)
    b = _params("bias", bias, N, dev)
    shape = x.shape[:-1] + (N,)
    ldr = 0
    if res is not None:
        _check("res", res, dev, (x.dtype,))
        if res.shape != shape:
            raise ValueError(f"res has shape {tuple(res.shape)}, expected {tuple(shape)}")
        ldr = _rows("res", res)[1]
    if out is None:
        out, ldo = x.new_empty(shape), N
    else:
        _check_out("out", out, shape, x, (x, weight, b), same=res)
        ldo = _rows("out", out)[1]
    pre = torch.empty_like(out, memory_format=torch.contiguous_format) if save_pre else None
    if M:
        lib = _lib.load()
        code = _TD[x.dtype]
        n = _linear_ws(False, code, M, K, N, order)
        ws = x.new_empty(n, dtype=torch.float32) if n > 0 else None
        _call(lib.ldm_linear, dev, code, x.data_ptr(), ldx, weight.data_ptr(), ldw, order, _data(b), _data(res), ldr,
              LINEAR_ACTS[act], out.data_ptr(), ldo, _data(pre), N, M, K, N, _data(ws))
    return (out, pre) if save_pre else out


def linear_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, pre: Optional[torch.Tensor] = None,
                    act: Optional[str] = None, dx: bool = True, dweight: bool = True, dbias: bool = True):
    """Gradients of linear (ldm_linear_backward): (dx, dweight, dbias, dz).  dz = dy act'(pre) is the gradient of the value
    before the activation and so of `res` (dy itself without an activation); dx = dz W^T; dweight = x^T dz, laid out like
    weight; dbias = column sums of dz, f32.  pre: linear's second output (save_pre), needed with an activation.
    dx, dweight or dbias False leaves that gradient out (None)."""
    dev, K, N = _check_linear(x, weight, act)
    shape = x.shape[:-1] + (N,)
    code_act = LINEAR_ACTS[act]
    if code_act and pre is None:
        raise ValueError("the gradient of an activation needs pre (linear's save_pre)")
    if not code_act:
        pre = None
    for name, t in (("dy", dy), ("pre", pre)):
        if t is not None or name == "dy":
            _check(name, t, dev, (x.dtype,))
            if t.shape != shape:
                raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    M, ldx = _rows("x", x)
    lddy = _rows("dy", dy)[1]
    ldp = 0 if pre is None else _rows("pre", pre)[1]
    order, ldw = _weight_order(weight)
    dz = _like(dy) if code_act else dy
    gx = _like(x) if dx else None
    gw = None
    if dweight:
        gw = _like(weight if order == 0 else weight.t())
    gb = x.new_empty(N, dtype=torch.float32) if dbias else None
    lib = _lib.load()
    code = _TD[x.dtype]
    n = _linear_ws(True, code, M, K, N, order)
    ws = x.new_empty(n, dtype=torch.float32) if n > 0 else None
    _call(lib.ldm_linear_backward, dev, code, dy.data_ptr(), lddy, x.data_ptr(), ldx, weight.data_ptr(), ldw, order,
          _data(pre), ldp, code_act, dz.data_ptr() if code_act else 0, N, _data(gx), K, _data(gw), N if order == 0 else K,
          _data(gb), _data(ws), M, K, N)
    return gx, (gw if gw is None or order == 0 else gw.t()), gb, dz
