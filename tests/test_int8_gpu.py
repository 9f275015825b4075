"""8-bit codes, products and the deformable convolution on them against their
64-bit forms.

The sums of codes are exact, so a float32 result is off by the roundings of the
two scales and the bias alone (3 * 2^-24 of the terms); 16 bits add half a step.
Codes made inside a call differ from the 64-bit ones only where a value lies so
near the middle of two codes that its fp32 error decides.  For given values
that is the division's: the codes equal those of the same fp32 division.  For
sampled columns some eight roundings of 2^-24 times 127 put at most 127 * 2^-20
= 1.3e-4 of the codes on the other side; one code in 1.3e-4 of a root mean
square of 20 and more is 6e-4 of a result."""
import ctypes

import pytest
import torch

import pytorch_mps_deform_conv2d_b200 as dcn
from _dense_ref import codes, deform_int8, rel
from pytorch_mps_deform_conv2d_b200 import _native
from pytorch_mps_deform_conv2d_b200.ops import STATUS_DENSE_TIMEOUT, TEST_WAIT_TIMEOUT

pytestmark = pytest.mark.gpu

FLIPS = 6e-4
FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rand_codes(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-128, 128, shape, device="cuda", dtype=torch.int8, generator=g)


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (5, 16), (3, 7, 33), (200, 768), (2, 4099), (1, 40000)],
                         ids=str)
def test_codes_are_those_of_the_formula(cuda_device, shape, dtype):
    torch.manual_seed(0)
    x = (torch.randn(shape, device="cuda") * torch.logspace(-3, 3, shape[-1], device="cuda")).to(dtype)
    q, s = dcn.quantize_int8(x)
    top = x.float().abs().amax(-1)
    assert torch.equal(s, top / torch.full_like(top, 127.0))
    assert torch.equal(q, torch.round(x.float() / s[..., None]).to(torch.int8))
    assert q.dtype == torch.int8 and q.shape == x.shape and s.shape == x.shape[:-1]


def test_code_corner_cases(cuda_device):
    x = torch.randn(6, 50, device="cuda")
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 8] = -float("inf")
    x[4] = torch.arange(50, device="cuda") * 0.5 - 0.5  # ties: scale is not 1 here
    x[5] = 0
    x[5, 0], x[5, 1], x[5, 2] = 127.0, 2.5, -3.5  # scale 1: ties go to even
    q, s = dcn.quantize_int8(x)
    assert s[1] == 0 and not q[1].any()
    assert s[2].isnan() and not q[2].any() and s[3].isinf() and not q[3].any()
    assert q[5, :3].tolist() == [127, 2, -4]
    strided = torch.randn(40, 64, device="cuda").t()
    assert torch.equal(dcn.quantize_int8(strided)[0], dcn.quantize_int8(strided.contiguous())[0])
    for shape in ((0, 4), (3, 0), (0,)):
        q, s = dcn.quantize_int8(torch.empty(shape, device="cuda"))
        assert q.shape == shape and s.shape == shape[:-1]


def linear_ref(q, xs, w, ws, b):
    y = (q.double() @ w.double().T) * xs.double()[..., None] * ws.double()
    return y if b is None else y + b.double()


def check_linear(got, q, xs, w, ws, b):
    want = linear_ref(q, xs, w, ws, b)
    size = linear_ref(q, xs, w, ws, None).abs() + (0 if b is None else b.double().abs())
    bound = 3.1 * 2.0 ** -24 * size + half_step(got.dtype) * want.abs()
    bound += torch.finfo(got.dtype).tiny  # results below the normal range
    assert got.shape == want.shape
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("out", FLOATS, ids=str)
@pytest.mark.parametrize("tokens,cin,cout", [(1, 16, 1), (1, 4096, 4096), (2, 160, 257), (7, 33, 5),
                                             (8, 1024, 130), (16, 2048, 512), (17, 512, 64),
                                             (64, 768, 1000), (130, 129, 131), (300, 1000, 700),
                                             (1025, 256, 640), (2500, 64, 2300)])
def test_products_of_codes(cuda_device, tokens, cin, cout, out):
    q, w = rand_codes(tokens, cin, seed=1), rand_codes(cout, cin, seed=2)
    torch.manual_seed(tokens)
    xs, ws = torch.rand(tokens, device="cuda"), torch.rand(cout, device="cuda") / cin
    b = torch.randn(cout, device="cuda").to(out) if tokens % 2 else None
    y = dcn.int8_linear(q, w, ws, b, x_scale=xs, out_dtype=out)
    assert y.dtype == out
    check_linear(y, q, xs, w, ws, b)
    assert dcn.device_status() == 0


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("shape,cout", [((1, 4096), 320), ((4, 96), 24), ((3, 5, 771), 1001),
                                        ((33, 1600), 96), ((700, 512), 512)], ids=str)
def test_floating_tokens(cuda_device, shape, cout, dtype):
    torch.manual_seed(1)
    x = torch.randn(shape, device="cuda").to(dtype)
    w, ws = rand_codes(cout, shape[-1], seed=3), torch.rand(cout, device="cuda") / shape[-1]
    b = torch.randn(cout, device="cuda")
    q, xs = dcn.quantize_int8(x)
    y = dcn.int8_linear(x, w, ws, b)
    assert y.dtype == dtype
    check_linear(y, q, xs, w, ws, b)


def test_longest_sums_fit(cuda_device):
    k = 131071
    q = torch.full((2, k), -128, dtype=torch.int8, device="cuda")
    one = torch.ones(2, device="cuda")
    y = dcn.int8_linear(q, q, one, x_scale=one)
    assert torch.equal(y, torch.full((2, 2), float(16384 * k), device="cuda"))
    with pytest.raises(RuntimeError, match="131071"):
        dcn.int8_linear(torch.zeros(1, k + 1, dtype=torch.int8, device="cuda"),
                        torch.zeros(1, k + 1, dtype=torch.int8, device="cuda"), one[:1],
                        x_scale=one[:1])


def test_offset_and_strided_operands(cuda_device):
    for tokens in (3, 140):
        base, wbase = rand_codes(tokens + 1, 96, seed=4), rand_codes(97, 96, seed=5)
        xs, ws = torch.rand(tokens, device="cuda"), torch.rand(96, device="cuda")
        # 32 bytes of a row further on, an odd address, rows of every other column
        for q, w in ((base[1:, 32:], wbase[1:, 32:]),
                     (base.flatten()[5:5 + tokens * 64].view(tokens, 64),
                      wbase.flatten()[3:3 + 96 * 64].view(96, 64)),
                     (base[1:, ::2], wbase[1:, ::2])):
            y = dcn.int8_linear(q, w, ws, x_scale=xs)
            check_linear(y, q, xs, w, ws, None)


def test_rows_that_are_not_finite_stay_in_their_rows(cuda_device):
    for tokens in (3, 200):
        x = torch.randn(tokens, 64, device="cuda")
        x[1, 5] = float("nan")
        x[2, 6] = float("inf")
        x[0] = 0
        y = dcn.int8_linear(x, rand_codes(48, 64), torch.rand(48, device="cuda"))
        assert y[1:3].isnan().all() and not y[0].any()
        assert tokens == 3 or y[3:].isfinite().all()


def test_linear_refusals_and_empty(cuda_device):
    q, w, s = rand_codes(4, 32), rand_codes(8, 32), torch.rand(8, device="cuda")
    xs = torch.rand(4, device="cuda")
    for args, kw, match in (((q, w, s), {}, "x_scale"),
                            ((xs.new_zeros(4, 32), w, s), dict(x_scale=xs), "x_scale"),
                            ((q, w, s), dict(x_scale=xs[:3]), "leading shape"),
                            ((q, w[:, :16], s), dict(x_scale=xs), "features"),
                            ((q, w, s[:7]), dict(x_scale=xs), "weight_scale"),
                            ((q, w, s.half()), dict(x_scale=xs), "weight_scale"),
                            ((q, w, s, s[:5]), dict(x_scale=xs), "bias"),
                            ((q, w.float(), s), dict(x_scale=xs), "int8"),
                            ((q.double(), w, s), {}, "x must be"),
                            ((q, w, s), dict(x_scale=xs, out_dtype=torch.int32), "out_dtype")):
        with pytest.raises(RuntimeError, match=match):
            dcn.int8_linear(*args, **kw)
    with pytest.raises(RuntimeError, match="no gradient"):
        dcn.int8_linear(xs.new_zeros(4, 32).requires_grad_(), w, s)
    assert dcn.int8_linear(q[:0], w, s, x_scale=xs[:0]).shape == (0, 8)
    assert dcn.int8_linear(q, w[:0], s[:0], x_scale=xs).shape == (4, 0)


# ---- the deformable convolution ----------------------------------------------------


def deform_case(n=2, c=16, h=9, w=11, o=12, kh=3, kw=3, stride=(1, 1), pad=(1, 1), dil=(1, 1),
                groups=1, dg=1, mask=True, bias=True, spread=2.0, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    ho = (h + 2 * pad[0] - dil[0] * (kh - 1) - 1) // stride[0] + 1
    wo = (w + 2 * pad[1] - dil[1] * (kw - 1) - 1) // stride[1] + 1
    wq = rand_codes(o, c // groups, kh, kw, seed=seed).contiguous(memory_format=torch.channels_last)
    return dict(x=rnd(n, c, h, w).to(dtype), off=(spread * rnd(n, 2 * dg * kh * kw, ho, wo)).to(dtype),
                wq=wq, ws=torch.rand(o, device="cuda", generator=g) / 100,
                bias=rnd(o).to(dtype) if bias else None,
                mask=torch.sigmoid(rnd(n, dg * kh * kw, ho, wo)).to(dtype) if mask else None,
                stride=stride, pad=pad, dil=dil)


def run_deform(k, **kw):
    return dcn.deform_conv2d_int8(k["x"], k["off"], k["wq"], k["ws"], k["bias"], k["stride"],
                                  k["pad"], k["dil"], k["mask"], **kw)


def ref_deform(k):
    return deform_int8(k["x"], k["off"], k["wq"], k["ws"], k["bias"], k["mask"], k["stride"],
                       k["pad"], k["dil"])


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("case", [
    dict(), dict(c=64, o=64, h=16, w=16), dict(c=256, o=256, n=1, h=20, w=23, spread=4.0),
    dict(kh=1, kw=1, pad=(0, 0), c=48, o=40), dict(kh=5, kw=3, pad=(2, 0), c=8, o=7),
    dict(stride=(2, 1), pad=(2, 1), dil=(2, 1), c=32, o=20, dg=8, mask=False, bias=False),
    dict(groups=2, dg=4, c=16, o=6), dict(groups=4, dg=2, c=24, o=8), dict(groups=16, c=16, o=16),
    dict(groups=3, dg=3, c=9, o=6), dict(c=1, o=1, n=1, h=1, w=1), dict(c=5, o=300, h=14, w=15),
    dict(n=5, c=20, h=31, w=7, o=130, spread=30.0), dict(c=96, dg=3, groups=2, o=10),
    dict(c=520, o=16, n=1, h=6, w=5), dict(c=8, o=9, spread=0.0),
    dict(c=40, dg=2, o=8), dict(c=40, dg=4, o=8), dict(c=24, groups=2, dg=1, o=4),
    dict(c=200, dg=10, kh=5, kw=5, pad=(2, 2), o=4), dict(c=260, dg=2, o=5),
    dict(c=1100, dg=4, n=1, h=5, w=6, o=4)], ids=str)
def test_deform_matches_64_bits(cuda_device, case, dtype):
    k = deform_case(**case, dtype=dtype)
    y = run_deform(k)
    assert y.dtype == dtype and y.is_contiguous()
    assert rel(y, ref_deform(k)) <= FLIPS + half_step(dtype)
    assert dcn.device_status() == 0


def test_deform_more_columns_than_shared_memory_holds(cuda_device):
    k = deform_case(n=1, c=6000, h=4, w=5, o=9)
    assert rel(run_deform(k), ref_deform(k)) <= FLIPS


def test_deform_layouts_and_types(cuda_device):
    k = deform_case(c=24, o=10, dtype=torch.float32)
    y = run_deform(k)
    for change in (dict(x=k["x"].contiguous(memory_format=torch.channels_last)),
                   dict(wq=k["wq"].contiguous()), dict(off=k["off"].mT.contiguous().mT),
                   dict(x=torch.cat([k["x"], k["x"]], 3)[..., :11])):
        assert torch.equal(run_deform({**k, **change}), y)
    for out in (torch.bfloat16, torch.float16):
        assert torch.equal(run_deform(k, out_dtype=out), y.to(out))
    logits = torch.randn_like(k["mask"])
    a = run_deform({**k, "mask": logits}, mask_logits=True)
    b = run_deform({**k, "mask": torch.sigmoid(logits)})
    assert rel(a, b) <= FLIPS


def test_deform_far_offsets_and_values_that_are_not_finite(cuda_device):
    k = deform_case(c=16, o=8, bias=False)
    k["off"] = torch.full_like(k["off"], 1e6)  # every sample outside: rows of zeros
    assert not run_deform(k).any()
    k = deform_case(n=2, c=16, o=8, spread=0.0)
    k["x"][1, 3, 4, 4] = float("nan")
    y = run_deform(k)
    assert y[0].isfinite().all() and y[1, :, 4, 4].isnan().all() and y[1, :, 8, 8].isfinite().all()


@pytest.mark.parametrize("c", [16, 5])
def test_deform_values_at_the_edges_of_the_range(cuda_device, c):
    # columns whose scale is below the normal range, and masks that are not
    # finite where nothing is sampled
    k = deform_case(c=c, o=8, bias=False)
    small = {**k, "x": k["x"] * 1e-38}
    assert rel(run_deform(small).double() * 1e30, ref_deform(small) * 1e30) <= 2e-2
    far = {**k, "off": torch.full_like(k["off"], 1e6),
           "mask": torch.full_like(k["mask"], float("nan"))}
    assert not run_deform(far).any()


def test_deform_in_several_chunks_of_pixels(cuda_device):
    # 2 x 78400 pixels of 2304 codes: more than are kept at a time.  Pixels do
    # not depend on one another: image by image gives the same bits
    k = deform_case(n=2, c=256, h=280, w=280, o=40, dtype=torch.bfloat16)
    y = run_deform(k)
    for i in range(2):
        one = {**k, **{t: k[t][i:i + 1] for t in ("x", "off", "mask")}}
        assert torch.equal(run_deform(one)[0], y[i])


def test_one_dimensional_token(cuda_device):
    x, w, s = torch.randn(64, device="cuda"), rand_codes(24, 64), torch.rand(24, device="cuda")
    assert torch.equal(dcn.int8_linear(x, w, s), dcn.int8_linear(x[None], w, s)[0])
    q, xs = dcn.quantize_int8(x)
    assert xs.shape == () and torch.equal(dcn.int8_linear(q, w, s, x_scale=xs),
                                          dcn.int8_linear(x, w, s))


def test_operators_under_compile_and_opcheck(cuda_device):
    x, w, s = torch.randn(6, 64, device="cuda"), rand_codes(24, 64), torch.rand(24, device="cuda")
    k = deform_case()

    def all_of(x):
        q, xs = dcn.quantize_int8(x)
        return (dcn.int8_linear(x, w, s), dcn.int8_linear(q, w, s, x_scale=xs),
                dcn.newton_schulz(x), run_deform(k))

    for a, b in zip(torch.compile(all_of, fullgraph=True, backend="aot_eager")(x), all_of(x)):
        assert torch.equal(a, b)
    ops = _native.load_ops()
    tests = ("test_schema", "test_faketensor")
    torch.library.opcheck(ops.quantize_int8.default, (x,), test_utils=tests)
    torch.library.opcheck(ops.int8_linear.default, (x, w, s), test_utils=tests)
    torch.library.opcheck(ops.newton_schulz.default, (x, 5, [3.4445, -4.775, 2.0315], 1e-7),
                          test_utils=tests)
    p, g, m = (torch.randn(8, 16, device="cuda") for _ in range(3))
    torch.library.opcheck(ops.muon_update_.default,
                          ([p], [g], [m], 0.1, 0.9, True, 0.0, 5, [3.4445, -4.775, 2.0315], 1e-7),
                          test_utils=tests)


def test_deform_refusals_and_empty(cuda_device):
    k = deform_case()
    for change, match in ((dict(off=k["off"][:, :, 1:]), "offset shape"),
                          (dict(mask=k["mask"][:, 1:]), "mask shape"),
                          (dict(off=k["off"].half()), "must both be"),
                          (dict(mask=k["mask"].half()), "type"),
                          (dict(wq=k["wq"].float()), "int8"),
                          (dict(ws=k["ws"][1:]), "weight_scale"),
                          (dict(bias=k["bias"][1:]), "bias"),
                          (dict(stride=(0, 1)), "stride"),
                          (dict(x=k["x"][:, :7]), "in-channels")):
        with pytest.raises(RuntimeError, match=match):
            run_deform({**k, **change})
    with pytest.raises(RuntimeError, match="no gradient"):
        run_deform({**k, "x": k["x"].requires_grad_()})
    e = deform_case(n=0)
    assert run_deform(e).shape == (0, 12, 9, 11)


def test_a_wait_that_runs_out_is_reported(cuda_device):
    dcn.device_status()
    q, w, s = rand_codes(200, 64), rand_codes(48, 64), torch.rand(48, device="cuda")
    xs = torch.rand(200, device="cuda")
    _native.load_ops().int8_linear(q, w, s, None, xs, None, TEST_WAIT_TIMEOUT)
    assert dcn.device_status() & STATUS_DENSE_TIMEOUT
    check_linear(dcn.int8_linear(q, w, s, x_scale=xs), q, xs, w, s, None)


def test_graphs_share_nothing(cuda_device):
    k1, k2 = deform_case(c=32, o=40), deform_case(c=64, o=24, h=15, seed=3, dtype=torch.bfloat16)
    x = torch.randn(5, 160, device="cuda")
    w, s = rand_codes(70, 160), torch.rand(70, device="cuda")
    calls = (lambda: run_deform(k1), lambda: run_deform(k2), lambda: dcn.int8_linear(x, w, s))
    for c in calls:
        c()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c())
        graphs.append(g)
    for _ in range(2):
        for t in (k1["x"], k2["x"], x):
            t.copy_(torch.randn_like(t))
        for g in reversed(graphs):
            g.replay()
        for c, o in zip(calls, outs):
            assert torch.equal(c(), o)


@pytest.mark.parametrize("modulated", [True, False])
def test_train_with_muon_then_serve_in_8_bits(cuda_device, modulated):
    torch.manual_seed(0)
    block = dcn.DeformConv2dPack(32, 48, 3, padding=1, deformable_groups=2, modulated=modulated).cuda()
    torch.nn.init.normal_(block.conv_offset.weight, std=0.05)
    opt = dcn.Muon([block.weight, block.conv_offset.weight], lr=0.02)
    rest = torch.optim.SGD([block.bias, block.conv_offset.bias], lr=0.02)
    x, y = torch.randn(2, 32, 14, 13, device="cuda"), torch.randn(2, 48, 14, 13, device="cuda")
    for _ in range(3):
        opt.zero_grad()
        rest.zero_grad()
        (block(x) - y).square().mean().backward()
        opt.step()
        rest.step()
    served = dcn.Int8DeformConv2d.from_float(block)
    q, s = codes(block.weight.detach().flatten(1))
    # the weight's fp32 division decides a code in some 127 * 2^-23
    assert (served.weight.flatten(1).double() - q).abs().sum() <= 2
    assert rel(served.weight_scale, s) <= 2.0 ** -23
    with torch.no_grad():
        om = block.conv_offset(x)
        want = deform_int8(x, om[:, :36], served.weight, served.weight_scale, served.bias,
                           torch.sigmoid(om[:, 36:].double()) if modulated else None, (1, 1), (1, 1),
                           (1, 1))
        assert rel(served(x), want) <= FLIPS
        # and near the float block: codes are off by half a step of max / 127
        assert rel(served(x), block(x)) <= 0.05
    clone = dcn.Int8DeformConv2d.from_float(block)
    clone.load_state_dict(served.state_dict())
    assert torch.equal(clone(x), served(x))
    plain = dcn.Int8DeformConv2d.from_float(dcn.DeformConv2d(8, 8, 3).cuda())
    with pytest.raises(TypeError, match="offset"):
        plain(torch.randn(1, 8, 5, 5, device="cuda"))


@pytest.mark.parametrize("tokens,cin,cout", [(4096, 64, 4096), (6000, 640, 3000), (40000, 64, 64)])
def test_waits_that_run_out_over_many_tiles_are_reported(cuda_device, tokens, cin, cout):
    # more tiles than CTAs: a CTA that gives up still walks through those it has left
    dcn.device_status()
    q, w, s = rand_codes(tokens, cin), rand_codes(cout, cin), torch.rand(cout, device="cuda")
    xs = torch.rand(tokens, device="cuda")
    _native.load_ops().int8_linear(q, w, s, None, xs, None, TEST_WAIT_TIMEOUT)
    assert dcn.device_status() & STATUS_DENSE_TIMEOUT
    check_linear(dcn.int8_linear(q, w, s, x_scale=xs), q, xs, w, s, None)
    dcn.check_device_status()


def test_rows_without_columns_have_scale_zero(cuda_device):
    lib = _native.load_capi()
    for t in range(3):  # DCN_TYPE_F32, BF16, F16
        s = torch.full((5,), 7.0, device="cuda")
        assert lib.dcn_quantize_int8(5, 0, t, None, None, s.data_ptr(),
                                     torch.cuda.current_stream().cuda_stream) == 0
        assert not s.any()


def test_a_served_pack_is_apart_from_the_trained_one(cuda_device):
    torch.manual_seed(0)
    block = dcn.DeformConv2dPack(16, 16, 3, padding=1).cuda()
    torch.nn.init.normal_(block.conv_offset.weight, std=0.1)
    served = dcn.Int8DeformConv2d.from_float(block)
    x = torch.randn(1, 16, 9, 9, device="cuda")
    y = served(x)
    with torch.no_grad():
        for p in block.parameters():
            p.add_(0.1)
    assert torch.equal(served(x), y)
    assert not any(p.requires_grad for p in served.parameters())
    served.half()
    assert {p.dtype for p in block.parameters()} == {torch.float32}
    assert all(p.requires_grad for p in block.parameters())
    assert served(x.half()).dtype == torch.half


@pytest.mark.parametrize("modulated", [True, False])
def test_gradients_are_refused_not_dropped(cuda_device, modulated):
    x = torch.randn(1, 8, 7, 7, device="cuda")
    leaf = x.clone().requires_grad_()
    block = dcn.DeformConv2dPack(8, 8, 3, padding=1, modulated=modulated).cuda()
    served = dcn.Int8DeformConv2d.from_float(block)
    plain = dcn.Int8DeformConv2d.from_float(dcn.DeformConv2d(8, 8, 3, padding=1).cuda())
    # (a conv_offset that asks for gradients, given by hand)
    own = dcn.Int8DeformConv2d(served.weight, served.weight_scale, served.bias, 1, 1, 1,
                               block.conv_offset, modulated=modulated)
    off = torch.zeros(1, 18, 7, 7, device="cuda")
    mask = torch.ones(1, 9, 7, 7, device="cuda")
    calls = (lambda: served(leaf), lambda: own(x), lambda: plain(leaf, off),
             lambda: plain(x, off.clone().requires_grad_()),
             lambda: plain(x, off, mask.clone().requires_grad_()),
             lambda: dcn.quantize_int8(block.weight.flatten(1)))
    for call in calls:
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
        with torch.no_grad():
            call()
    with torch.no_grad():
        assert torch.equal(own(x), served(leaf))
    assert not served(x).requires_grad


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("h,w", [(0, 5), (5, 0), (0, 0)])
def test_images_without_pixels_answer_with_the_bias(cuda_device, h, w, dtype):
    # all padding, as deform_conv2d takes them
    torch.manual_seed(0)
    x = torch.empty(2, 4, h, w, device="cuda", dtype=dtype)
    off = torch.randn(2, 18, h + 2, w + 2, device="cuda").to(dtype)
    mask, b = torch.rand(2, 9, h + 2, w + 2, device="cuda").to(dtype), torch.randn(6, device="cuda")
    wq, ws = rand_codes(6, 4, 3, 3), torch.rand(6, device="cuda")
    want = b.to(dtype)[None, :, None, None].expand(2, 6, h + 2, w + 2)
    got = dcn.deform_conv2d_int8(x, off, wq, ws, b, padding=2, mask=mask)
    assert torch.equal(got, want)
    if dtype == torch.float32:
        assert torch.equal(dcn.deform_conv2d(x, off, wq.float(), b, padding=2, mask=mask), want)
    # the C entry point, told that they lie channels last
    lib = _native.load_capi()
    s = _native.DcnShape(batch=2, in_channels=4, height=h, width=w, out_channels=6, kernel_h=3,
                         kernel_w=3, stride_h=1, stride_w=1, pad_h=2, pad_w=2, dilation_h=1,
                         dilation_w=1, groups=1, deformable_groups=1)
    t, flags = FLOATS.index(dtype), 0x20000  # DCN_INPUT_NHWC
    out = torch.empty_like(got)
    ws_bytes = lib.dcn_deform_int8_workspace_size(ctypes.byref(s), t, flags)
    space = torch.empty(ws_bytes, dtype=torch.uint8, device="cuda")
    wl = wq.permute(0, 2, 3, 1).contiguous()
    assert lib.dcn_deform_int8(ctypes.byref(s), t, None, wl.data_ptr(), ws.data_ptr(), off.data_ptr(),
                               mask.data_ptr(), b.data_ptr(), 0, out.data_ptr(), t, flags,
                               space.data_ptr(), ws_bytes,
                               torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out, want)


@pytest.mark.parametrize("given", [True, False])
@pytest.mark.parametrize("cin,cout", [(64, 40), (1024, 96), (2304, 250), (4096, 1000), (4096, 8200)])
def test_two_to_nine_tokens_by_either_way(cuda_device, cin, cout, given):
    # one kernel, or coder and tensor-core product, by sizes; without a workspace
    # the former up to eight
    lib = _native.load_capi()
    w, ws = rand_codes(cout, cin, seed=1), torch.rand(cout, device="cuda") / cin
    for tokens in range(2, 10):
        x = torch.randn(tokens, cin, device="cuda").bfloat16()
        q, xs = dcn.quantize_int8(x)
        kw = dict(x_scale=xs) if given else {}
        y = dcn.int8_linear(q if given else x, w, ws, out_dtype=torch.float32, **kw)
        check_linear(y, q, xs, w, ws, None)
        if tokens <= 8:
            z = torch.empty_like(y)
            a, t, s = (q, 3, xs.data_ptr()) if given else (x, 1, None)
            assert lib.dcn_int8_linear(tokens, cin, cout, t, a.data_ptr(), s, w.data_ptr(),
                                       ws.data_ptr(), None, 0, z.data_ptr(), 0, 0, None, 0,
                                       torch.cuda.current_stream().cuda_stream) == 0
            check_linear(z, q, xs, w, ws, None)


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16], ids=str)
def test_waits_that_run_out_in_clusters_are_reported(cuda_device, out):
    # few tiles, K split over a cluster whose partial sums never come
    dcn.device_status()
    q, w, s = rand_codes(20, 4096), rand_codes(250, 4096), torch.rand(250, device="cuda")
    xs = torch.rand(20, device="cuda")
    _native.load_ops().int8_linear(q, w, s, None, xs, out, TEST_WAIT_TIMEOUT)
    assert dcn.device_status() & STATUS_DENSE_TIMEOUT
    check_linear(dcn.int8_linear(q, w, s, x_scale=xs, out_dtype=out), q, xs, w, s, None)
    dcn.check_device_status()
