"""newton_schulz, muon_update_ and Muon against their 64-bit forms.

Tolerances (2-norms, relative).  fp32: operands of two fp16 terms are off by at
most 2^-23 and a product's sums by about as much; some twenty products enter a
result, and five steps multiply an early error by up to 40 where the singular
values near 1 keep moving (|x p'(x) / p(x)| up to 2 a step): 20 * 2^-23 * 40 /
sqrt(40) -- errors of the products are independent -- is below 2e-5.  16-bit
results: half a step of the type, eps / 2, plus for bf16 the one rounding of X
to fp16 (2^-11) two steps from the end, times a^2 = 11.9 (in single steps X, S
and P are rounded, each by 2^-12 at most where the largest values lie and 2^-13 in
the mean: no more than that one in three steps together)."""
import ctypes

import pytest
import torch

import pytorch_mps_deform_conv2d_b200 as dcn
from _dense_ref import COEF, muon, orthogonalise, rel
from pytorch_mps_deform_conv2d_b200 import _native
from pytorch_mps_deform_conv2d_b200.ops import STATUS_DENSE_TIMEOUT, TEST_WAIT_TIMEOUT

pytestmark = pytest.mark.gpu

F32 = 2e-5
TOL = {torch.float32: F32, torch.float16: 2.0 ** -11 + F32,
       torch.bfloat16: 2.0 ** -8 + 11.9 * 2.0 ** -11}
DTYPES = sorted(TOL, key=str)


def gradient(*shape, dtype=torch.float32, seed=0):
    """A few strong directions over noise."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, cols = shape[-2:]
    r = max(1, min(rows, cols) // 16)
    lead = shape[:-2]
    u = torch.randn(*lead, rows, r, device="cuda", generator=g)
    v = torch.randn(*lead, r, cols, device="cuda", generator=g)
    return (1e-3 * (u @ v / r ** 0.5 + 0.3 * torch.randn(*shape, device="cuda", generator=g))).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(16, 16), (1, 1), (1, 33), (33, 1), (64, 576), (65, 127),
                                   (127, 65), (128, 128), (129, 1000), (1000, 129), (256, 2304),
                                   (515, 300), (3, 40, 72), (2, 3, 130, 50), (70, 8, 18)], ids=str)
def test_matches_64_bits(cuda_device, shape, dtype):
    x = gradient(*shape, dtype=dtype, seed=len(shape))
    before = x.clone()
    y = dcn.newton_schulz(x)
    assert y.dtype == dtype and y.shape == x.shape and y.is_contiguous()
    assert torch.equal(x, before)
    assert rel(y, orthogonalise(x)) <= TOL[dtype]
    assert dcn.device_status() == 0


@pytest.mark.parametrize("shape", [(1100, 2051), (2051, 1100), (4096, 512), (700, 1000), (1000, 700),
                                   (520, 520)], ids=str)
def test_many_tiles(cuda_device, shape):
    for dtype in DTYPES:
        x = gradient(*shape, dtype=dtype)
        assert rel(dcn.newton_schulz(x), orthogonalise(x)) <= TOL[dtype], dtype


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 11])
def test_steps(cuda_device, steps):
    # a cubic that settles: errors are not multiplied for ever
    coef = (1.5, -0.5, 0.0)
    for shape in ((48, 100), (100, 48)):
        x = gradient(*shape)
        got = dcn.newton_schulz(x, steps=steps, coefficients=coef)
        assert rel(got, orthogonalise(x, steps, coef)) <= F32


def test_coefficients_a_step(cuda_device):
    coef = [(3.4445, -4.7750, 2.0315), (4.0, -6.0, 2.6), (1.875, -1.25, 0.375), (1.5, -0.5, 0.0)]
    x = gradient(72, 200)
    assert rel(dcn.newton_schulz(x, steps=4, coefficients=coef), orthogonalise(x, 4, coef)) <= F32


def test_tf32_mode_keeps_11_bits(cuda_device):
    x = gradient(256, 640)
    dcn.set_math_mode("tf32")
    try:
        y = dcn.newton_schulz(x)
    finally:
        dcn.set_math_mode(None)
    # X is rounded to fp16 (2^-11) at the start and once between: a^5 and a^3 at
    # most of it reaches the smallest directions, a^2 the whole
    assert rel(y, orthogonalise(x)) <= 2 * 11.9 * 2.0 ** -11


def test_strided_inputs(cuda_device):
    base = gradient(3, 96, 160)
    for x in (base.mT, base[:, ::2, 1::3], base[1:, 5:, 7:], base.expand(2, 3, 96, 160)):
        assert rel(dcn.newton_schulz(x), orthogonalise(x)) <= F32


def test_scale_of_the_input(cuda_device):
    x = gradient(40, 64)
    for scale in (1e-30, 1e-12, 1e30):  # 1e-30: far below eps, the answer is as small
        assert rel(dcn.newton_schulz(x * scale, eps=1e-37), orthogonalise(x * scale, eps=1e-37)) <= F32
    tiny = x * 1e-9  # the norm is about eps
    assert rel(dcn.newton_schulz(tiny), orthogonalise(tiny)) <= F32


def test_zeros_and_values_that_are_not_finite(cuda_device):
    for dtype in DTYPES:
        x = gradient(4, 48, 80, dtype=dtype)
        x[0] = 0
        x[1, 3, 5] = float("nan")
        x[2, 7, 0] = float("inf")
        y = dcn.newton_schulz(x)
        assert torch.equal(y[0], torch.zeros_like(y[0]))
        assert y[1].isnan().all() and y[2].isnan().all()
        assert rel(y[3], orthogonalise(x[3])) <= TOL[dtype]
    z = gradient(60, 60)
    z[10:20] = 0  # rows of zeros stay zero
    y = dcn.newton_schulz(z)
    assert torch.equal(y[10:20], torch.zeros_like(y[10:20])) and rel(y, orthogonalise(z)) <= F32


def test_empty(cuda_device):
    for shape in ((0, 5), (5, 0), (0, 4, 4)):
        assert dcn.newton_schulz(torch.empty(shape, device="cuda")).shape == shape


def test_same_bits_again_and_on_another_stream(cuda_device):
    x = gradient(300, 700)
    a = dcn.newton_schulz(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = dcn.newton_schulz(x)
        c = dcn.newton_schulz(x * 2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b) and c.isfinite().all()


def test_two_graphs_and_an_eager_call(cuda_device):
    xs = [gradient(96, 300, seed=1), gradient(640, 200, seed=2, dtype=torch.bfloat16)]
    for x in xs:
        dcn.newton_schulz(x)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(dcn.newton_schulz(x))
        graphs.append(g)
    for seed in (5, 6):
        for x in xs:
            x.copy_(gradient(*x.shape, dtype=x.dtype, seed=seed))
        graphs[1].replay()
        graphs[0].replay()
        for x, o in zip(xs, outs):
            assert torch.equal(o, dcn.newton_schulz(x))


def test_refusals(cuda_device):
    x = gradient(8, 8)
    with pytest.raises(RuntimeError, match="at least two dimensions"):
        dcn.newton_schulz(x[0])
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        dcn.newton_schulz(x.double())
    with pytest.raises(RuntimeError, match="steps must be"):
        dcn.newton_schulz(x, steps=0)
    with pytest.raises(RuntimeError, match="triple"):
        dcn.newton_schulz(x, coefficients=(1.0, 2.0))
    with pytest.raises(RuntimeError, match="at most 15"):
        dcn.newton_schulz(x, coefficients=(16.0, 0.0, 0.0))
    with pytest.raises(RuntimeError, match="at most 15"):
        dcn.newton_schulz(x, coefficients=(float("nan"), 0.0, 0.0))
    with pytest.raises(RuntimeError, match="no gradient"):
        dcn.newton_schulz(x.requires_grad_())


def test_a_wait_that_runs_out_is_reported(cuda_device):
    dcn.device_status()
    x = gradient(64, 64)
    _native.load_ops().newton_schulz(x, 5, list(COEF), 1e-7, TEST_WAIT_TIMEOUT)
    assert dcn.device_status() & STATUS_DENSE_TIMEOUT
    assert rel(dcn.newton_schulz(x), orthogonalise(x)) <= F32
    dcn.check_device_status()


# ---- the optimiser step ---------------------------------------------------------
# A new parameter: (1 - lr wd) p - lr s o, three fp32 roundings and lr s |o| times
# the error above; 16 bits add half a step.  Momentum: three fp32 roundings.


def leaves(shapes, dtype=torch.float32, seed=0, fmt=torch.contiguous_format):
    ps, gs, ms = [], [], []
    for i, s in enumerate(shapes):
        rows, cols = s[0], int(torch.Size(s).numel() / s[0])
        for out, sd, dt in ((ps, 1, dtype), (gs, 2, dtype), (ms, 3, torch.float32)):
            t = gradient(rows, cols, dtype=dt, seed=100 * seed + 10 * i + sd).reshape(s)
            t = 50 * t if out is ps else t
            out.append(t.contiguous(memory_format=fmt) if len(s) == 4 else t.contiguous())
    return ps, gs, ms


def check_step(ps, gs, ms, **kw):
    want = [muon(p, g, m, **{k.replace("adjust", "match_rms"): v == "match_rms" if k == "adjust"
                             else v for k, v in kw.items()}) for p, g, m in zip(ps, gs, ms)]
    dcn.muon_update_(ps, gs, ms, **kw)
    for p, m, (wp, wm) in zip(ps, ms, want):
        half = torch.finfo(p.dtype).eps / 2
        update = float((wp - p.double()).norm())
        err = float((p.double() - wp).norm())
        o = kw["lr"] * max(p.shape) ** 0.5 * 3
        assert err <= (half + 3 * 2.0 ** -24) * float(wp.norm()) + TOL[p.dtype] * o, (err, update)
        assert rel(m, wm) <= 3 * 2.0 ** -24


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_muon_step(cuda_device, dtype, nesterov):
    shapes = [(64, 16, 3, 3), (16, 64, 1, 1), (130, 50), (64, 16, 3, 3), (7, 3, 5, 5)]
    ps, gs, ms = leaves(shapes, dtype)
    check_step(ps, gs, ms, lr=0.02, nesterov=nesterov, weight_decay=0.1, momentum=0.9)


def test_muon_groups_scales_and_many_tensors(cuda_device):
    check_step(*leaves([(64, 2, 3, 3), (32, 8, 3, 3)]), lr=0.05, groups=32)
    check_step(*leaves([(96, 40), (40, 96)]), lr=0.05, adjust="match_rms")
    check_step(*leaves([(8, 16)] * 70), lr=0.05)
    check_step(*leaves([(256, 256, 3, 3)] * 2), lr=0.02, momentum=0.0)


def test_muon_takes_channels_last_weights_and_gradients_of_other_layouts(cuda_device):
    ps, gs, ms = leaves([(24, 12, 3, 3)], fmt=torch.channels_last)
    check_step(ps, gs, ms, lr=0.02)
    ps, gs, ms = leaves([(24, 12, 3, 3), (31, 17)])
    gs[0] = gs[0].contiguous(memory_format=torch.channels_last)
    gs[1] = gs[1].t().contiguous().t()
    check_step(ps, gs, ms, lr=0.02)


def test_muon_refusals(cuda_device):
    ps, gs, ms = leaves([(8, 16)])
    for kw, match in (
            (dict(params=ps, grads=gs, momenta=[]), "as many"),
            (dict(params=ps * 2, grads=gs * 2, momenta=ms * 2), "twice"),
            (dict(params=ps, grads=[gs[0].half()], momenta=ms), "same type"),
            (dict(params=ps, grads=gs, momenta=[ms[0].half()]), "momenta must be float32"),
            (dict(params=ps, grads=[gs[0][:4]], momenta=ms), "shape"),
            (dict(params=[ps[0].t()], grads=[gs[0].t()], momenta=[ms[0].t()]), "outermost"),
            (dict(params=ps, grads=gs, momenta=ms, groups=3), "divisible"),
            (dict(params=ps, grads=gs, momenta=ms, momentum=1.0), "momentum")):
        before = ps[0].clone()
        with pytest.raises(RuntimeError, match=match):
            dcn.muon_update_(lr=0.1, **kw)
        assert torch.equal(ps[0], before)


def test_muon_refuses_overlapping_views(cuda_device):
    whole, state = torch.randn(12, 16, device="cuda"), torch.zeros(2, 8, 16, device="cuda")
    g = torch.randn(8, 16, device="cuda")
    with pytest.raises(RuntimeError, match="overlap"):
        dcn.muon_update_([whole[:8], whole[4:]], [g, g], list(state), lr=0.1)
    dcn.muon_update_([whole[:4], whole[4:]], [g[:4], g], [state[0, :4], state[1]], lr=0.1)


def test_muon_bumps_versions(cuda_device):
    ps, gs, ms = leaves([(8, 16)])
    w = ps[0].requires_grad_()
    y = (w * w).sum()
    dcn.muon_update_(ps, gs, ms, lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def make_layer(seed=0, groups=1):
    torch.manual_seed(seed)
    return dcn.DeformConv2d(16, 24, 3, padding=1, groups=groups).cuda()


def test_optimizer_trains_a_layer(cuda_device):
    torch.manual_seed(0)
    layer = make_layer(groups=4)
    opt = dcn.Muon([dict(params=[layer.weight], groups=4)], lr=0.02, weight_decay=0.01)
    x = torch.randn(2, 16, 12, 12, device="cuda")
    off, m = torch.randn(2, 18, 12, 12, device="cuda"), torch.rand(2, 9, 12, 12, device="cuda")
    momentum = torch.zeros(24, 4, 3, 3, device="cuda")
    for _ in range(3):
        opt.zero_grad()
        layer(x, off, m).square().mean().backward()
        w, g = layer.weight.detach().clone(), layer.weight.grad.clone()
        opt.step()
        want, momentum = muon(w, g, momentum, lr=0.02, weight_decay=0.01, groups=4)
        got = layer.weight.detach().double()
        assert float((got - want).norm()) <= 4 * 2.0 ** -24 * float(want.norm()) + F32 * 0.02 * 24
        momentum = opt.state[layer.weight]["momentum_buffer"].clone()


def test_optimizer_state_survives_a_checkpoint(cuda_device):
    p = torch.nn.Parameter(gradient(32, 48, dtype=torch.bfloat16))
    q = torch.nn.Parameter(p.detach().clone())
    a, b = dcn.Muon([p], lr=0.1), dcn.Muon([q], lr=0.1)
    p.grad = gradient(32, 48, dtype=torch.bfloat16, seed=1)
    a.step()
    q.data.copy_(p.data)
    b.load_state_dict(a.state_dict())
    assert b.state[q]["momentum_buffer"].dtype == torch.float32
    assert torch.equal(a.state[p]["momentum_buffer"], b.state[q]["momentum_buffer"])
    p.grad = q.grad = gradient(32, 48, dtype=torch.bfloat16, seed=2)
    a.step()
    b.step()
    assert torch.equal(p, q)
    assert a.state[p]["momentum_buffer"].data_ptr() != b.state[q]["momentum_buffer"].data_ptr()


def test_optimizer_step_in_a_graph(cuda_device):
    layer, twin = make_layer(1), make_layer(1)
    opts = [dcn.Muon([m.weight], lr=0.02) for m in (layer, twin)]
    g = [gradient(24, 144, seed=s).reshape(24, 16, 3, 3) for s in range(4)]
    layer.weight.grad, twin.weight.grad = g[0].clone(), g[0].clone()
    for o in opts:  # makes the state before the capture
        o.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opts[0].step()
    for s in (1, 2, 3):
        layer.weight.grad.copy_(g[s])
        twin.weight.grad.copy_(g[s])
        graph.replay()
        opts[1].step()
    assert torch.equal(layer.weight, twin.weight)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_waits_that_run_out_over_many_tiles_are_reported(cuda_device, dtype):
    dcn.device_status()
    x = gradient(6, 700, 900, dtype=dtype)
    _native.load_ops().newton_schulz(x, 5, list(COEF), 1e-7, TEST_WAIT_TIMEOUT)
    assert dcn.device_status() & STATUS_DENSE_TIMEOUT
    assert rel(dcn.newton_schulz(x), orthogonalise(x)) <= TOL[dtype]
    dcn.check_device_status()


@pytest.mark.parametrize("eps", [1e-7, 1e-20, 1e-37, 0.0])
@pytest.mark.parametrize("shape", [(2, 48, 80), (2, 80, 48), (2, 150, 200), (2, 200, 500)], ids=str)
def test_zeros_stay_zero_whatever_eps_is(cuda_device, shape, eps):
    # (1 / eps and its square leave fp32's range)
    for dtype in DTYPES:
        x = gradient(*shape, dtype=dtype)
        x[0] = 0
        y = dcn.newton_schulz(x, eps=eps)
        assert torch.equal(y[0], torch.zeros_like(y[0]))
        assert rel(y[1], orthogonalise(x[1], eps=eps)) <= TOL[dtype]


@pytest.mark.parametrize("eps", [1e-7, 1e-20, 0.0])
def test_muon_leaves_a_layer_without_updates_alone(cuda_device, eps):
    for shape in ((24, 40), (150, 200)):
        ps, gs, ms = leaves([shape] * 2)
        gs[0].zero_()
        ms[0].zero_()
        before = ps[0].clone()
        dcn.muon_update_(ps, gs, ms, lr=0.1, eps=eps)
        assert torch.equal(ps[0], before) and not ms[0].any() and ps[1].isfinite().all()


@pytest.mark.parametrize("tf32", [False, True])
def test_a_last_run_of_one_step_on_few_directions(cuda_device, tf32):
    # Two runs of one step (13^2 ends the first).  S is 0.7327 in the first, where
    # fp16 leaves a low term of 2^-13, and 2.9e-4 in the second, whose polynomial
    # 0.01 + 15 S would take a quarter of its value from a low term of the first.
    # p(S) of the first, 0.02, is the difference of terms of 13 to 2^-22: 2e-4
    coef, eps = [(13.0, -15.0, -3.7072), (0.01, 15.0, 0.0)], 0.67312
    x = torch.ones(1, 16, device="cuda", dtype=torch.float32 if tf32 else torch.bfloat16)
    if tf32:
        dcn.set_math_mode("tf32")
    try:
        y = dcn.newton_schulz(x, steps=2, coefficients=coef, eps=eps)
    finally:
        dcn.set_math_mode(None)
    assert rel(y, orthogonalise(x, 2, coef, eps)) <= TOL[torch.bfloat16]


@pytest.mark.parametrize("steps", [4, 6, 7, 10])
@pytest.mark.parametrize("shape", [(64, 576), (100, 48), (128, 300), (200, 900)], ids=str)
def test_steps_of_16_bit_results(cuda_device, shape, steps):
    # 4, 7 and 10 steps end in a run of one
    for dtype in (torch.bfloat16, torch.float16):
        x = gradient(*shape, dtype=dtype)
        assert rel(dcn.newton_schulz(x, steps=steps), orthogonalise(x, steps)) <= TOL[dtype]


def fp16_between(u, coef, squares):
    """The choice made for bf16 results, in 64 bits: X as one fp16 term between
    single steps, with `squares` S and P of all but the first two as well."""
    def half(x, scale):
        return (x * scale).half().double() / scale

    x = u.double() / (u.double().norm() + 1e-7)
    flip = x.shape[0] > x.shape[1]
    x = x.mT if flip else x
    for i, (a, b, c) in enumerate(coef):
        cut = (lambda t: half(t, 1024.0)) if squares and i > 1 else (lambda t: t)
        s = cut(x @ x.mT)
        p = cut(a * torch.eye(len(s), dtype=s.dtype, device=s.device) + b * s + c * (s @ s))
        x = p @ x
        if i + 1 < len(coef):
            x = half(x, 1024.0)
    return x.mT if flip else x


@pytest.mark.parametrize("coef,squares", [([COEF] * 5, True), ([(4.125, -11.75, 8.5)] * 5, False),
                                          ([(4.5, -14.0, 10.0)] * 4, False)], ids=str)
@pytest.mark.parametrize("shape", [(300, 500), (520, 520), (700, 400)], ids=str)
def test_bf16_results_are_off_by_the_roundings_chosen_for_them(cuda_device, shape, coef, squares):
    # Those of X, S and P, and the result's own, are independent: their squares
    # add.  A quarter more for where the roundings fall.  (S and P keep two terms
    # for coefficients that would multiply their roundings.)
    x = gradient(*shape, dtype=torch.bfloat16)
    want = orthogonalise(x, len(coef), coef)
    chosen, own = rel(fp16_between(x, coef, squares), want), rel(want.bfloat16(), want)
    got = dcn.newton_schulz(x, steps=len(coef), coefficients=coef)
    assert rel(got, want) <= (own ** 2 + (1.25 * chosen) ** 2) ** 0.5


@pytest.mark.parametrize("shape", [(2304, 2304), (2570, 2304), (2304, 7000)], ids=str)
def test_products_of_sm_pairs_with_mirrored_halves(cuda_device, shape):
    # Gram matrices from some 2200 rows take 256 x 256 tiles on two SMs and write
    # both halves: one-term squares for bf16 (two terms where X is long), two for
    # float16
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x = gradient(*shape, dtype=dtype)
        want = orthogonalise(x)
        bound = TOL[dtype]
        if dtype == torch.bfloat16:
            chosen, own = rel(fp16_between(x, [COEF] * 5, True), want), rel(want.bfloat16(), want)
            bound = (own ** 2 + (1.25 * chosen) ** 2) ** 0.5
        assert rel(dcn.newton_schulz(x), want) <= bound, dtype
    assert dcn.device_status() == 0


@pytest.mark.parametrize("shape", [(64, 576), (200, 300), (300, 900), (900, 300)], ids=str)
def test_schedules_of_steep_polynomials(cuda_device, shape):
    # first steps whose b and c are beyond 15; singular values stay below 2.  Errors
    # of S reach P times |b| + 2 |c| = 58 in the first step, 9 at most in the others
    # and in the usual schedule: 6.5 times its bound for float32
    coef = [(8.25, -23.5, 17.0), (4.1, -2.95, 0.545), (3.95, -2.9, 0.55), (3.3, -2.45, 0.5),
            (2.3, -1.65, 0.42)]
    for dtype in DTYPES:
        x = gradient(*shape, dtype=dtype)
        bound = 6.5 * F32 + (0 if dtype == torch.float32 else TOL[dtype])
        assert rel(dcn.newton_schulz(x, coefficients=coef), orthogonalise(x, 5, coef)) <= bound


def test_muon_refuses_grads_that_it_would_write(cuda_device):
    whole, p, g = (torch.randn(24, 16, device="cuda") for _ in range(3))
    before, held = p.clone(), g.clone()
    z = torch.zeros_like(p)
    for params, grads, momenta in (([p], [g], [g]), ([p], [p], [z]), ([p, g], [z, p], [whole, z[:]]),
                                   ([p, whole[:8]], [g, whole[7:15]], [z, z.new_zeros(8, 16)]),
                                   ([whole[8:16]], [whole[1:24:3]], [z.new_zeros(8, 16)])):
        with pytest.raises(RuntimeError, match="overlap"):
            dcn.muon_update_(params, grads, momenta, lr=0.1)
    assert torch.equal(p, before) and torch.equal(g, held)
    # neighbours, and one gradient for two
    dcn.muon_update_([whole[:8], whole[16:]], [whole[8:16]] * 2, list(z.new_zeros(2, 8, 16)), lr=0.1)


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("momentum", [0.0, 0.3, 0.99, 0.999, 0.99999])
def test_muon_weighs_the_gradient_by_one_minus_momentum(cuda_device, momentum, nesterov):
    # from a momentum of zeros: (1 - momentum) g, two roundings
    ps, gs, _ = leaves([(24, 40), (150, 200)])
    ms = [torch.zeros_like(p) for p in ps]
    check_step(ps, gs, ms, lr=0.02, momentum=momentum, nesterov=nesterov)


def test_muon_c_entry_points_agree(cuda_device):
    lib = _native.load_capi()
    c = (ctypes.c_float * 3)(*COEF)
    ws_bytes = lib.dcn_muon_update_workspace_size(1, 24, 40, 0, 1, 0)
    space = torch.empty(ws_bytes, dtype=torch.uint8, device="cuda")
    got = []
    for fn in (lib.dcn_muon_update, lib.dcn_muon_update_f64):
        (p,), (g,), (m,) = leaves([(24, 40)])
        one = lambda t: (ctypes.c_void_p * 1)(t.data_ptr())  # noqa: E731
        # settings that float holds
        assert fn(1, 24, 40, 0, one(p), one(g), one(m), 0.25, 0.875, 1, 0.5, 1.5, 1, c, 1e-7, 0,
                  space.data_ptr(), ws_bytes, torch.cuda.current_stream().cuda_stream) == 0
        got.append((p, m))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_muon_refuses_a_size_before_it_writes_anything(cuda_device):
    side = 32769  # both sides: beyond what is supported
    small = torch.randn(8, 16, device="cuda", dtype=torch.bfloat16)
    large = torch.empty(side, side, device="cuda", dtype=torch.bfloat16)
    ps, ms = [small, large], [torch.zeros_like(p, dtype=torch.float32) for p in (small, large)]
    gs = [torch.ones_like(small), small.new_ones(1).expand(side, side)]
    before = small.clone()
    with pytest.raises(RuntimeError, match="not supported"):
        dcn.muon_update_(ps, gs, ms, lr=0.1)
    assert torch.equal(small, before) and not ms[0].any()


def test_the_first_step_is_not_captured(cuda_device):
    # a graph that held the momentum's zeros would start from them in every replay
    w = torch.nn.Parameter(gradient(24, 40))
    w.grad = gradient(24, 40, seed=1)
    opt = dcn.Muon([w], lr=0.1)
    before = w.detach().clone()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    dcn.newton_schulz(w.detach())  # (the kernels are loaded)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph.capture_begin()
        with pytest.raises(RuntimeError, match="before the one"):
            opt.step()
        spare = torch.zeros(1, device="cuda")  # something to capture
        graph.capture_end()
    assert torch.equal(w, before) and not opt.state and spare is not None
    opt.step()
    assert opt.state[w]["momentum_buffer"].any() and not torch.equal(w, before)
