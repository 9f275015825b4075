"""Host-side behaviour of the orthogonalised updates and 8-bit products: no
fallback on the CPU, refusals of the C entry points before anything is
launched, shape inference of the operators."""
import ctypes

import pytest
import torch

import pytorch_mps_deform_conv2d_b200 as dcn
from pytorch_mps_deform_conv2d_b200 import _native

F32, BF16, F16, I8 = range(4)
OK, INVALID, WORKSPACE, CUDA, UNSUPPORTED = range(5)
P = 1 << 20  # an address that is never read: every call below is refused on the host


def test_cpu_tensors_are_refused():
    x, q, s = torch.randn(4, 16), torch.zeros(4, 16, dtype=torch.int8), torch.ones(4)
    for call in (lambda: dcn.newton_schulz(x), lambda: dcn.muon_update_([x], [x], [x], lr=0.1),
                 lambda: dcn.quantize_int8(x), lambda: dcn.int8_linear(x, q, s),
                 lambda: dcn.deform_conv2d_int8(torch.randn(1, 2, 5, 5), torch.zeros(1, 18, 3, 3),
                                                torch.zeros(2, 2, 3, 3, dtype=torch.int8), s[:2])):
        with pytest.raises(NotImplementedError, match="CUDA"):
            call()


def test_optimizer_arguments():
    w = torch.nn.Parameter(torch.randn(6, 4))
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(adjust="none")):
        with pytest.raises(ValueError):
            dcn.Muon([w], **kw)
    with pytest.raises(ValueError, match="two dimensions"):
        dcn.Muon([torch.nn.Parameter(torch.randn(6))])
    with pytest.raises(ValueError, match="divisible"):
        dcn.Muon([dict(params=[w], groups=4)])
    with pytest.raises(ValueError, match="divisible"):
        dcn.Muon([w], groups=0)
    opt = dcn.Muon([w])
    assert opt.step() is None  # nothing has a gradient: nothing is called
    with pytest.raises(ValueError, match="adjust"):
        dcn.muon_update_([w], [w], [w], lr=0.1, adjust="x")


def coef(*v):
    return (ctypes.c_float * len(v))(*v)


def test_newton_schulz_c_refusals():
    lib = _native.load_capi()
    c = coef(3.4, -4.8, 2.0)
    ws = lib.dcn_newton_schulz_workspace_size(1, 64, 128, F32, 1, 0)
    assert ws > 0 and lib.dcn_newton_schulz_workspace_size(1, 64, 128, I8, 1, 0) == 0
    assert lib.dcn_newton_schulz_workspace_size(1, 64, 128, F32, 33, 0) == 0

    def call(count=1, rows=64, cols=128, t=F32, x=P, out=P, steps=1, co=c, eps=0.0, n=ws, w=P):
        return lib.dcn_newton_schulz(count, rows, cols, t, x, out, steps, co, eps, 0, w, n, None)

    assert call(n=ws - 1) == WORKSPACE and call(w=None) == WORKSPACE
    assert call(x=None) == INVALID and call(out=None) == INVALID and call(co=None) == INVALID
    assert call(t=I8) == INVALID and call(steps=0) == INVALID and call(eps=-1.0) == INVALID
    assert call(rows=-1) == INVALID and call(co=coef(1e9, 0, 0)) == INVALID
    assert call(rows=1 << 16, cols=1 << 15) == UNSUPPORTED
    assert call(rows=40000, cols=40000) == UNSUPPORTED
    assert call(count=0) == OK and call(rows=0) == OK
    assert b"dcn_newton_schulz" in (call(x=None), lib.dcn_last_error())[1]


def test_muon_c_refusals():
    lib = _native.load_capi()
    c = coef(3.4, -4.8, 2.0)
    vp = ctypes.c_void_p
    some, none = (vp * 1)(P), (vp * 1)(None)
    ws = lib.dcn_muon_update_workspace_size(1, 64, 128, BF16, 1, 0)

    def call(p=some, g=some, m=some, momentum=0.9, n=ws, t=BF16):
        return lib.dcn_muon_update(1, 64, 128, t, p, g, m, 0.1, momentum, 1, 0.0, 1.0, 1, c, 1e-7, 0,
                                   P, n, None)

    assert call(p=none) == INVALID and call(g=none) == INVALID and call(m=none) == INVALID
    assert call(p=None) == INVALID and call(momentum=1.0) == INVALID and call(t=I8) == INVALID
    assert call(n=ws - 1) == WORKSPACE


def test_int8_c_refusals():
    lib = _native.load_capi()
    assert lib.dcn_quantize_int8(2, 8, I8, P, P, P, None) == INVALID
    assert lib.dcn_quantize_int8(2, 8, F32, None, P, P, None) == INVALID
    assert lib.dcn_quantize_int8(1 << 31, 8, F32, P, P, P, None) == UNSUPPORTED
    assert lib.dcn_quantize_int8(0, 8, F32, None, None, None, None) == OK
    ws = lib.dcn_int8_linear_workspace_size(4, 64, 32, F16)
    assert ws > 0 and lib.dcn_int8_linear_workspace_size(0, 64, 32, F16) == 0

    def call(tokens=4, cin=64, cout=32, t=F16, x=P, xs=None, w=P, sc=P, b=None, bt=F32, o=P, ot=F16,
             n=ws):
        return lib.dcn_int8_linear(tokens, cin, cout, t, x, xs, w, sc, b, bt, o, ot, 0, P, n, None)

    assert call(xs=P) == INVALID and call(t=I8) == INVALID  # x_scale with int8 and only then
    assert call(x=None) == INVALID and call(w=None) == INVALID and call(sc=None) == INVALID
    assert call(o=None) == INVALID and call(ot=I8) == INVALID and call(b=P, bt=I8) == INVALID
    assert call(cin=0) == INVALID and call(cin=131072) == UNSUPPORTED
    assert call(n=ws - 1) == WORKSPACE and call(tokens=0) == OK
    # without a workspace: only a few tokens, of whole and aligned rows
    none = lambda tokens, cin, w: lib.dcn_int8_linear(  # noqa: E731
        tokens, cin, 32, F16, P, None, w, P, None, F32, P, F16, 0, None, 0, None)
    assert none(9, 64, P) == WORKSPACE and none(4, 63, P) == WORKSPACE
    assert none(4, 64, P + 1) == WORKSPACE


def test_deform_int8_c_refusals():
    lib = _native.load_capi()
    good = dict(batch=1, in_channels=4, height=6, width=6, out_channels=4, kernel_h=3, kernel_w=3,
                stride_h=1, stride_w=1, pad_h=1, pad_w=1, dilation_h=1, dilation_w=1, groups=1,
                deformable_groups=1)

    def call(t=F32, x=P, n=1 << 30, ot=F32, **kw):
        s = _native.DcnShape(**{**good, **kw})
        return lib.dcn_deform_int8(ctypes.byref(s), t, x, P, P, P, None, None, F32, P, ot, 0, P, n,
                                   None)

    assert call(n=16) == WORKSPACE and call(x=None) == INVALID and call(t=I8) == INVALID
    assert call(ot=I8) == INVALID and call(stride_h=0) == INVALID and call(groups=3) == INVALID
    assert call(in_channels=20000) == UNSUPPORTED  # 180000 columns a group
    assert call(batch=65536) == UNSUPPORTED
    assert call(batch=0) == OK


def test_int8_module_keeps_its_scales_in_float32():
    m = dcn.Int8DeformConv2d(torch.zeros(4, 2, 3, 3, dtype=torch.int8), torch.rand(4),
                             torch.rand(4), 1, 1, 1)
    scale = m.weight_scale.clone()
    m = m.half()
    assert m.weight.dtype == torch.int8 and m.bias.dtype == torch.float16
    assert m.weight_scale.dtype == torch.float32 and torch.equal(m.weight_scale, scale)
    assert set(m.state_dict()) == {"weight", "weight_scale", "bias"}


def meta(*shape, dtype=torch.float32):
    return torch.empty(*shape, device="meta", dtype=dtype)


def test_operators_infer_shapes():
    ops = _native.load_ops()
    y = ops.newton_schulz(meta(3, 8, 4, dtype=torch.bfloat16), 5, [1.0, 0.0, 0.0], 1e-7)
    assert y.shape == (3, 8, 4) and y.dtype == torch.bfloat16
    q, s = ops.quantize_int8(meta(3, 5, 8))
    assert q.shape == (3, 5, 8) and q.dtype == torch.int8 and s.shape == (3, 5)
    w = meta(6, 8, dtype=torch.int8)
    assert ops.int8_linear(meta(2, 3, 8, dtype=torch.half), w, meta(6)).dtype == torch.half
    y = ops.int8_linear(meta(2, 8, dtype=torch.int8), w, meta(6), None, meta(2))
    assert y.shape == (2, 6) and y.dtype == torch.float32
    y = ops.deform_conv2d_int8(meta(2, 4, 9, 9), meta(6, 4, 3, 3, dtype=torch.int8), meta(6),
                               meta(2, 18, 9, 9), None, None, 1, 1, 1, 1, 1, 1, 1, 1,
                               torch.bfloat16)
    assert y.shape == (2, 6, 9, 9) and y.dtype == torch.bfloat16


def test_sides_that_tiles_would_round_past_31_bits_are_refused():
    # the last refused by its workspace: the size itself is taken
    lib = _native.load_capi()
    c, top = coef(3.4, -4.8, 2.0), (1 << 31) - 256

    def schulz(rows, cols):
        return lib.dcn_newton_schulz(1, rows, cols, F32, P, P, 1, c, 0.0, 0, P, 16, None)

    def linear(tokens, cout):
        return lib.dcn_int8_linear(tokens, 16, cout, I8, P, P, P, P, None, F32, P, F32, 0, P, 16,
                                   None)

    def deform(cout):
        s = _native.DcnShape(batch=1, in_channels=1, height=1, width=1, out_channels=cout,
                             kernel_h=1, kernel_w=1, stride_h=1, stride_w=1, pad_h=0, pad_w=0,
                             dilation_h=1, dilation_w=1, groups=1, deformable_groups=1)
        return lib.dcn_deform_int8(ctypes.byref(s), F32, P, P, P, P, None, None, F32, P, F32, 0, P,
                                   16, None)

    for call in (lambda n: schulz(1, n), lambda n: schulz(n, 1), lambda n: linear(n, 1),
                 lambda n: linear(1, n), deform):
        assert call(top + 1) == UNSUPPORTED and call((1 << 31) - 1) == UNSUPPORTED
        assert call(top) == WORKSPACE
    for n in (top + 1, (1 << 31) - 1):
        assert lib.dcn_newton_schulz_workspace_size(1, 1, n, F32, 1, 0) == 0
        assert lib.dcn_muon_update_workspace_size(1, n, 1, F32, 1, 0) == 0


def test_int8_module_refuses_gradients():
    m = dcn.Int8DeformConv2d(torch.zeros(4, 2, 3, 3, dtype=torch.int8), torch.rand(4), None, 1, 1, 1)
    x, off = torch.randn(1, 2, 5, 5, requires_grad=True), torch.zeros(1, 18, 5, 5)
    with pytest.raises(RuntimeError, match="no gradient"):
        m(x, off)
    with torch.no_grad(), pytest.raises(NotImplementedError, match="CUDA"):
        m(x, off)


def test_polynomials_that_fit_are_taken():
    # by the values on [0, 1], whatever b and c are (the last refused by its workspace)
    lib = _native.load_capi()

    def call(*abc):
        return lib.dcn_newton_schulz(1, 64, 128, F32, P, P, 1, coef(*abc), 0.0, 0, P, 16, None)

    for abc in ((8.25, -23.5, 17.0), (15, 15, 15), (15, -30, 0), (-15, 30, 0), (0, 60, -60),
                (15, -120, 120)):
        assert call(*abc) == WORKSPACE, abc
    inf, nan = float("inf"), float("nan")
    for abc in ((15.1, 0, 0), (-16, 20, 0), (15, 16, 0), (0, 64, -64), (15, -125, 125), (3, 0, 20),
                (1, inf, 0), (1, -inf, inf), (1, nan, 0), (1, 0, nan), (3, 1e38, -1e38)):
        assert call(*abc) == INVALID, abc
    assert b"at most 15" in lib.dcn_last_error()


def test_few_tokens_query():
    few = _native.load_capi().dcn_int8_linear_few_tokens
    assert few(1, 4096, 1 << 20, BF16) == 1 and few(2, 8192, 8192, I8) == 1
    assert few(2, 4096, 4096, F16) == 1 and few(2, 8192, 8192, F16) == 0
    assert few(4, 1024, 4096, BF16) == 1 and few(4, 4096, 4096, BF16) == 0
    assert few(8, 4096, 4096, I8) == 1 and few(8, 4096, 4096, F32) == 0
    # rows that the kernel does not take, more tokens, nothing
    assert few(1, 4095, 16, BF16) == 0 and few(9, 64, 64, I8) == 0 and few(0, 64, 64, I8) == 0
