"""Operators of transformer blocks, CPU side: the C ABI refuses bad arguments before anything is launched, and the Python
surface's reading of shapes, strides and overlaps."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from diffusionmodel_amd import _lib
    return _lib.load()


P = C.c_void_p(4096)            # never dereferenced: every call below is refused on the host
BF, F32 = 1, 0


def _ln(lib, dtype=F32, x=P, xs=8, eps=1e-5, y=P, ys=8, rows=4, Cc=8):
    return lib.ldm_layer_norm(dtype, x, xs, None, None, eps, y, ys, None, None, rows, Cc, None)


def test_layer_norm_arguments(lib):
    for kw in (dict(dtype=2), dict(rows=-1), dict(Cc=0), dict(Cc=(1 << 24) + 1), dict(eps=-1.0), dict(eps=float("nan")),
               dict(x=None), dict(y=None), dict(ys=7), dict(xs=-8)):
        assert _ln(lib, **kw) == 1, kw
        assert b"layer_norm" in lib.ldm_last_error()
    assert _ln(lib, rows=0, x=None, y=None) == 0
    bwd = lambda dy=P, dxs=8, dw=P, db=P, ws=P, mean=P, rows=4: lib.ldm_layer_norm_backward(   # noqa: E731
        BF, dy, 8, P, 8, None, 0, mean, P, None, P, dxs, dw, db, ws, rows, 8, None)
    for kw in (dict(dy=None), dict(dxs=7), dict(dw=None), dict(db=None), dict(ws=None), dict(mean=None), dict(rows=-1)):
        assert bwd(**kw) == 1, kw
    assert lib.ldm_layer_norm_ws_floats(2, 4, 8) < 0 and lib.ldm_layer_norm_ws_floats(F32, 4, 0) < 0
    assert lib.ldm_layer_norm_ws_floats(F32, 0, 8) == 0
    for rows in (1, 5, 1000, 10 ** 9):
        for cc in (1, 8, 1000, 20000):
            assert 0 < lib.ldm_layer_norm_ws_floats(BF, rows, cc) <= 2 * 1024 * cc


def test_rope_arguments(lib):
    import struct

    def call(dtype=BF, q=P, k=P, oq=P, ok=P, st=struct.pack("12l", *([8] * 12)), B=1, N=4, Hq=2, Hk=1, D=8, pos=P, pt=0,
             ps=struct.pack("3l", 0, 4, 1), inv=P, sec=(2, 2), axes=None):
        axes = len(sec) if axes is None else axes
        return lib.ldm_rope(dtype, q, k, oq, ok, st, B, N, Hq, Hk, D, pos, pt, ps, inv,
                            None if sec is None else struct.pack(f"{len(sec)}i", *sec), axes, 0, 0, None)
    for kw in (dict(dtype=3), dict(q=None), dict(k=None), dict(oq=None), dict(ok=None), dict(st=None), dict(B=-1), dict(N=-1),
               dict(Hq=0), dict(Hk=-1), dict(D=0), dict(D=2049), dict(pos=None), dict(pt=3), dict(ps=None), dict(inv=None),
               dict(sec=(2, 3)), dict(sec=(5, -1)), dict(sec=(0, 0)), dict(sec=(1,) * 5), dict(sec=(2,), axes=0),
               dict(sec=None, axes=1), dict(B=65536, N=65536), dict(Hq=60000, Hk=6000)):
        assert call(**kw) == 1, kw
    assert call(B=0, q=None, k=None) == 0 and call(N=0) == 0


def test_linear_arguments(lib):
    def fwd(dtype=BF, x=P, w=P, order=0, act=0, out=P, ldo=16, pre=None, ldp=16, M=4, K=8, N=16, ldx=8):
        return lib.ldm_linear(dtype, x, ldx, w, 16, order, None, None, 0, act, out, ldo, pre, ldp, M, K, N, P, None)
    for kw in (dict(dtype=2), dict(x=None), dict(w=None), dict(out=None), dict(order=2), dict(act=4), dict(act=-1),
               dict(ldo=15), dict(pre=P, ldp=15), dict(M=-1), dict(K=0), dict(N=0), dict(K=1 << 30), dict(M=1 << 40),
               dict(ldx=-1)):
        assert fwd(**kw) == 1, kw
        assert b"linear" in lib.ldm_last_error()
    assert fwd(M=0, x=None) == 0

    def bwd(dy=P, x=P, w=P, act=0, pre=None, dz=None, lddz=16, dx=P, lddx=8, dw=P, lddw=16, db=P, ws=P, M=4, order=0):
        return lib.ldm_linear_backward(BF, dy, 16, x, 8, w, 16, order, pre, 16, act, dz, lddz, dx, lddx, dw, lddw, db, ws, M,
                                       8, 16, None)
    for kw in (dict(dy=None), dict(x=None), dict(w=None), dict(act=1), dict(act=1, pre=P), dict(act=1, dz=P),
               dict(act=1, pre=P, dz=P, lddz=15), dict(lddx=7), dict(lddw=15), dict(order=1, lddw=7), dict(ws=None),
               dict(M=-1)):
        assert bwd(**kw) == 1, kw
    assert lib.ldm_linear_ws_floats(2, 1, 1, 1, 0) < 0 and lib.ldm_linear_backward_ws_floats(BF, 1, 0, 1, 0) < 0
    for M, K, N in ((0, 1, 1), (1, 256, 2048), (65536, 4096, 1024), (16384, 1024, 4096), (10 ** 7, 64, 64)):
        for order in (0, 1):
            n = lib.ldm_linear_ws_floats(BF, M, K, N, order), lib.ldm_linear_backward_ws_floats(BF, M, K, N, order)
            assert min(n) >= 0 and max(n) * 4 < (1 << 30), (M, K, N, n)


def test_rows_of_strided_tensors():
    from diffusionmodel_amd import ops
    x = torch.zeros(4, 6, 30)
    assert ops._rows("x", x) == (24, 30)
    assert ops._rows("x", x[..., 5:15]) == (24, 30)
    assert ops._rows("x", x[1:3, :, :7]) == (12, 30)
    assert ops._rows("x", x[:, 0]) == (4, 180)
    assert ops._rows("x", x[:1].expand(4, 6, 30)[:, 0]) == (4, 0)
    assert ops._rows("x", torch.zeros(30).expand(5, 3, 30)) == (15, 0)
    assert ops._rows("x", torch.zeros(7)) == (1, 7)
    assert ops._rows("x", x[:0, :, :7]) == (0, 7)
    for bad in (x[:, :5], x.transpose(0, 1), x.transpose(1, 2), x[..., ::2], torch.zeros(1).expand(4, 3),
                x[:1].expand(4, 6, 30)):
        with pytest.raises(ValueError):
            ops._rows("x", bad)


def test_overlap_of_slices():
    from diffusionmodel_amd import ops
    qkv = torch.zeros(2, 5, 12, 8)
    q, k = qkv[:, :, :4], qkv[:, :, 4:8]
    assert ops._apart(q, k) and ops._apart(k, q) and ops._apart(qkv[0], qkv[1])
    assert not ops._apart(q, qkv) and not ops._apart(qkv[:, :, 2:6], k) and not ops._apart(q, q)
    heads_first = torch.zeros(2, 12, 5, 8).transpose(1, 2)
    assert ops._apart(heads_first[:, :, :4], heads_first[:, :, 4:]) and not ops._apart(heads_first[:, :, :5], heads_first[:, :, 4:])
    x = torch.zeros(6, 30)
    assert ops._apart(x[:, :10], x[:, 10:20]) and not ops._apart(x[:, :11], x[:, 10:20]) and not ops._apart(x[:4], x[1:5])
    assert ops._apart(x[:0], x)


def test_weight_orders():
    from diffusionmodel_amd import ops
    w = torch.zeros(8, 16)
    assert ops._weight_order(w) == (0, 16) and ops._weight_order(w.t()) == (1, 16)
    assert ops._weight_order(w[:, 3:9]) == (0, 16) and ops._weight_order(w[:, :1]) == (0, 16)
    assert ops._weight_order(w[:1].t()) == (0, 1) and ops._weight_order(w[:1]) == (0, 16)
    with pytest.raises(ValueError):
        ops._weight_order(torch.zeros(8, 8, 2)[..., 0])


def test_rope_frequencies():
    from diffusionmodel_amd import ops
    f = ops.rope_frequencies((2, 0, 4), theta=100.0)
    want = [1.0, 0.1] + [100.0 ** (-j / 4) for j in range(4)]
    assert f.dtype == torch.float32 and torch.allclose(f.double(), torch.tensor(want, dtype=torch.float64), rtol=1e-7)
    f = ops.rope_frequencies((2, 2), theta=100.0, shared=True)
    assert torch.allclose(f.double(), torch.tensor([100.0 ** (-j / 4) for j in range(4)], dtype=torch.float64), rtol=1e-7)
    for bad in ((), (0,), (2, -1)):
        with pytest.raises(ValueError):
            ops.rope_frequencies(bad)
    with pytest.raises(ValueError):
        ops.rope_frequencies((2,), theta=0.0)


def test_host_tensors_are_refused():
    from diffusionmodel_amd import ops
    x = torch.zeros(4, 8)
    for f in (lambda: ops.layer_norm(x), lambda: ops.linear(x, torch.zeros(8, 8)),
              lambda: ops.rope(torch.zeros(1, 2, 1, 8), None, torch.zeros(1, 2, dtype=torch.int32), torch.ones(4))):
        with pytest.raises(ValueError):
            f()


def test_launches_beyond_the_grid_are_refused(lib):
    import struct
    assert lib.ldm_linear(BF, P, 1, P, 1, 0, None, None, 0, 0, P, 1, None, 1, 1 << 36, 1, 1, P, None) == 1
    assert lib.ldm_linear(F32, P, 16, P, 1 << 29, 0, None, None, 0, 0, P, 1 << 29, None, 1, 4, 16, 1 << 29, P, None) == 1
    assert lib.ldm_linear_backward(F32, P, 1, P, 1, P, 1, 0, None, 0, 0, None, 0, None, 0, P, 1, None, P, 1 << 39, 1, 1,
                                   None) == 1
    assert lib.ldm_rope(F32, P, None, P, None, struct.pack("12l", *([2048] * 12)), 32768, 65535, 1, 0, 2048, P, 0,
                        struct.pack("3l", 0, 4, 1), P, struct.pack("i", 1024), 1, 0, 0, None) == 1


def test_what_torch_keeps_beside_the_memory_is_refused():
    """Forward-mode tangents and negated views have a data pointer like any tensor; the values would be misread."""
    from torch.autograd import forward_ad
    from diffusionmodel_amd import ops
    x = torch.randn(4, 8)
    ops._check_bits("x", x)
    with pytest.raises(ValueError, match="resolve_neg"):
        ops._check_bits("x", torch._neg_view(x))
    ops._check_bits("x", torch._neg_view(x).resolve_neg())
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        ops._check_bits("x", x)
        for t in (dual, dual[1:], dual.view(-1)):
            with pytest.raises(ValueError, match="tangent"):
                ops._check_bits("x", t)
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                ops._check("x", t)
        ops._check_bits("x", forward_ad.unpack_dual(dual).primal)


def test_sizes_beyond_32_bits_are_refused():
    """The C ABI's int arguments would take the low 32 bits: 2^32 + 8 columns would be 8."""
    from diffusionmodel_amd import ops
    for n in (2 ** 32 + 8, 2 ** 31, 2 ** 24 + 1, 0):
        with pytest.raises(ValueError, match="last axis"):
            ops._columns(torch.empty(1, n, device="meta"))
    with pytest.raises(ValueError, match="last axis"):
        ops._columns(torch.empty((), device="meta"))
    assert ops._columns(torch.empty(3, 1 << 24, device="meta")) == 1 << 24

    def plan(B, N, H, D):
        st = (N * H * D, H * D, D, 1)
        return ops._rope_plan((B, N, H, D), st, None, None, st, None, (1, N), (N, 1), 4, (4,), "half")
    assert plan(2, 3, 4, 8)[1] == (2, 3, 4, 0, 8)
    for dims in ((2 ** 32 + 1, 1, 1, 8), (1, 2 ** 32 + 5, 1, 8), (1, 1, 2 ** 32 + 1, 8), (1, 1, 1, 2 ** 32 + 8), (1, 2 ** 31, 1, 8)):
        with pytest.raises(ValueError, match="2\\^31"):
            plan(*dims)
