"""Timed cases of the operators around a deformable layer's weight matrix.

Training: ``newton_schulz`` (orthogonalising an update) and ``muon_update_``
(the optimiser step that uses it).  Serving: ``int8_linear`` (products of
8-bit integers with a scale for each token and each channel) and
``deform_conv2d_int8`` (the deformable convolution on such products).

``run`` computes each operator in its plain form, from elementary torch
operations, or with ``own`` set through the package's public entry points.
"""
import torch

own = False

#: The Newton-Schulz quintic x -> a x + b x^3 + c x^5 and the guard of the norm.
A, B, C = 3.4445, -4.7750, 2.0315
EPS = 1e-7
#: The optimiser's settings.
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # the update of the detection neck's layer: weight (256, 256, 3, 3) as a matrix
        dict(name="ns neck f32", op="ns", batch=1, rows=256, cols=2304, dtype="float32"),
        # a square projection of a large model, bf16 training
        dict(name="ns square bf16", op="ns", batch=1, rows=4096, cols=4096, dtype="bfloat16"),
        # ragged, more rows than columns, a few at once
        dict(name="ns tall odd f16", op="ns", batch=3, rows=1153, cols=515, dtype="float16"),
        # one small layer: latency
        dict(name="muon small f32", op="muon", layers=1, out=64, cin=64, k=3, nesterov=True, dtype="float32"),
        # the layers of a neck in one step
        dict(name="muon neck stack f32", op="muon", layers=6, out=256, cin=256, k=3, nesterov=True, dtype="float32"),
        # the 512-channel layers of the sweep, bf16 parameters, plain momentum
        dict(name="muon sweep bf16", op="muon", layers=4, out=512, cin=512, k=3, nesterov=False, dtype="bfloat16"),
        # one token through a square projection: decoding
        dict(name="linear one token bf16", op="linear", tokens=1, cin=4096, out=4096, bias=False, given=False, dtype="bfloat16"),
        # ragged in every direction, tokens quantised by the call
        dict(name="linear ragged f16", op="linear", tokens=197, cin=771, out=1001, bias=True, given=False, dtype="float16"),
        # a large batch of tokens that are in 8 bits already
        dict(name="linear batch i8 bf16", op="linear", tokens=8192, cin=4096, out=8192, bias=True, given=True, dtype="bfloat16"),
        # a small image, float32 in, bf16 out
        dict(name="deform small f32", op="deform", n=2, cin=64, h=16, w=16, out=64, k=3, s=1, p=1, d=1, groups=1, dg=1, mask=True, bias=True, spread=2.0, dtype="float32"),
        # the detection neck
        dict(name="deform neck bf16", op="deform", n=2, cin=256, h=100, w=152, out=256, k=3, s=1, p=1, d=1, groups=1, dg=1, mask=True, bias=True, spread=4.0, dtype="bfloat16"),
        # the DCNv1 sweep: 512 channels, 8 deformable groups, no mask
        dict(name="deform sweep f16", op="deform", n=64, cin=512, h=28, w=28, out=512, k=3, s=2, p=2, d=2, groups=1, dg=8, mask=False, bias=False, spread=3.0, dtype="float16"),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(("ns", "muon", "linear", "deform"))
    dtype = rng.choice(tuple(_DTYPES))
    if op == "ns":
        rows, cols = _log(rng, 16, 3000), _log(rng, 16, 3000)
        return dict(op=op, batch=rng.choice((1, 1, 2, 3, 5)), rows=rows, cols=cols, dtype=dtype)
    if op == "muon":
        return dict(op=op, layers=rng.randint(1, 6), out=_log(rng, 16, 512), cin=_log(rng, 4, 512), k=rng.choice((1, 3, 3, 5)),
                    nesterov=rng.random() < 0.5, dtype=rng.choice(("float32", "bfloat16")))
    if op == "linear":
        return dict(op=op, tokens=_log(rng, 1, 8192), cin=_log(rng, 16, 4096), out=_log(rng, 16, 8192), bias=rng.random() < 0.5,
                    given=rng.random() < 0.5, dtype=rng.choice(("bfloat16", "float16")))
    groups, dg = rng.choice((1, 1, 1, 2, 4)), rng.choice((1, 1, 2, 4))
    return dict(op=op, n=rng.randint(1, 4), cin=8 * _log(rng, 1, 40), h=_log(rng, 9, 90), w=_log(rng, 9, 90), out=groups * _log(rng, 4, 300 // groups),
                k=rng.choice((1, 3, 3, 5)), s=rng.choice((1, 1, 2)), p=rng.choice((1, 2)), d=1, groups=groups, dg=dg, mask=rng.random() < 0.7,
                bias=rng.random() < 0.5, spread=round(0.5 + 4 * rng.random(), 2), dtype=dtype)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _gradients(g, batch, rows, cols):
    """Matrices as gradients are: a few strong directions over broad noise."""
    r = max(1, min(rows, cols) // 16)
    strong = _randn(g, batch, rows, r) * torch.linspace(1.0, 0.1, r, device="cuda") @ _randn(g, batch, r, cols) / r**0.5
    return 1e-3 * (strong + 0.3 * _randn(g, batch, rows, cols))


def _out_size(c):
    size = lambda x: (x + 2 * c["p"] - c["d"] * (c["k"] - 1) - 1) // c["s"] + 1  # noqa: E731
    return size(c["h"]), size(c["w"])


def _weights_8bit(w):
    """An 8-bit weight with a scale for each row, as a program keeps it after loading."""
    scale = w.abs().amax(1) / 127.0
    return torch.round(w / scale[:, None]).clamp(-127, 127).to(torch.int8), scale


def prepare(case, seed):
    g, t = _gen(seed), _DTYPES[case["dtype"]]
    if case["op"] == "ns":
        return dict(case, x=_gradients(g, case["batch"], case["rows"], case["cols"]).to(t))
    if case["op"] == "muon":
        n, o, i, k = case["layers"], case["out"], case["cin"], case["k"]
        w = (i * k * k) ** -0.5 * _randn(g, n, o, i, k, k)
        grad = _gradients(g, n, o, i * k * k).view(n, o, i, k, k)
        buf = 0.7 * grad + 0.3 * _gradients(g, n, o, i * k * k).view(n, o, i, k, k)
        # separate tensors, as a model's parameters are; the momentum is float32 whatever they are
        return dict(case, p=[x.clone() for x in w.to(t)], g=[x.clone() for x in grad.to(t)], m=[x.clone() for x in buf])
    if case["op"] == "linear":
        m, n, k = case["tokens"], case["out"], case["cin"]
        wq, ws = _weights_8bit(_randn(g, n, k) * k**-0.5)
        # activations: channels of unlike size
        x = _randn(g, m, k) * torch.exp(0.7 * _randn(g, k))
        b = _randn(g, n).to(t) if case["bias"] else None
        if case["given"]:
            xq, xs = _weights_8bit(x)
            return dict(case, x=xq, xs=xs, wq=wq, ws=ws, b=b)
        return dict(case, x=x.to(t), xs=None, wq=wq, ws=ws, b=b)
    n, ci, o, k, gr, dg = case["n"], case["cin"], case["out"], case["k"], case["groups"], case["dg"]
    ho, wo = _out_size(case)
    wq, ws = _weights_8bit(_randn(g, o, ci // gr * k * k) * (ci // gr * k * k) ** -0.5)
    return dict(case, x=_randn(g, n, ci, case["h"], case["w"]).to(t), off=(case["spread"] * _randn(g, n, 2 * dg * k * k, ho, wo)).to(t),
                mk=torch.sigmoid(_randn(g, n, dg * k * k, ho, wo)).to(t) if case["mask"] else None,
                b=_randn(g, o).to(t) if case["bias"] else None, ws=ws,
                # the package's layout of a quantised weight: channels last, laid out once
                wq=wq.view(o, ci // gr, k, k).contiguous(memory_format=torch.channels_last))


# ---- the plain forms ----------------------------------------------------------


def _quintic(x):
    s = x @ x.mT
    return A * x + (B * s + C * (s @ s)) @ x


def _orthogonal(x):
    """Five Newton-Schulz steps over the smaller side, in 32 bits."""
    x = x.float()
    x = x / (x.double().square().sum((-2, -1), keepdim=True).sqrt() + EPS).float()
    if x.shape[-2] > x.shape[-1]:
        return _quintic(_quintic(_quintic(_quintic(_quintic(x.mT))))).mT
    return _quintic(_quintic(_quintic(_quintic(_quintic(x)))))


def _plain_muon(s):
    p, g, m = torch.stack(s["p"]), torch.stack(s["g"]).float(), torch.stack(s["m"])
    m = MOMENTUM * m + (1 - MOMENTUM) * g
    u = (1 - MOMENTUM) * g + MOMENTUM * m if s["nesterov"] else m
    rows, cols = s["out"], s["cin"] * s["k"] ** 2
    o = _orthogonal(u.flatten(2)).view_as(u)
    p = ((1 - LR * DECAY) * p.float() - LR * max(1.0, rows / cols) ** 0.5 * o).to(p.dtype)
    torch._foreach_copy_(s["p"], list(p))
    torch._foreach_copy_(s["m"], list(m))
    return {"p": s["p"], "m": s["m"]}


def _codes(x):
    """Rows of `x` as whole numbers of [-127, 127] and their scales."""
    top = x.abs().amax(-1, keepdim=True)
    scale = top / torch.full_like(top, 127.0)
    return torch.where(scale > 0, torch.round(x / scale), torch.zeros_like(x)), scale


def _plain_linear(s):
    q, scale = (s["x"].float(), s["xs"][:, None]) if s["given"] else _codes(s["x"].float())
    y = (q @ s["wq"].float().T) * scale * s["ws"]
    return (y if s["b"] is None else y + s["b"].float()).to(_DTYPES[s["dtype"]])


def _corner(img, y, x, h, w):
    """Values of img (N, dg, C / dg, H * W) at whole positions (N, dg, 1, taps * pixels); zero outside."""
    inside = (y >= 0) & (y < h) & (x >= 0) & (x < w)
    at = y.clamp(0, h - 1) * w + x.clamp(0, w - 1)
    return torch.gather(img, 3, at.long().expand(-1, -1, img.shape[2], -1)) * inside


def _columns(s, real):
    """Sampled columns (N, C, k * k, pixels) in the type `real`."""
    n, ci, h, w, k, dg = s["n"], s["cin"], s["h"], s["w"], s["k"], s["dg"]
    ho, wo = _out_size(s)
    grid = lambda size, taps: torch.arange(size, device="cuda", dtype=real) * s["s"] - s["p"] + taps * s["d"]  # noqa: E731
    taps = torch.arange(k, device="cuda", dtype=real)[:, None]
    off = s["off"].to(real).view(n, dg, k, k, 2, ho, wo)
    y = (off[:, :, :, :, 0] + grid(ho, taps)[:, None, :, None]).reshape(n, dg, 1, -1)
    x = (off[:, :, :, :, 1] + grid(wo, taps)[None, :, None, :]).reshape(n, dg, 1, -1)
    img = s["x"].to(real).view(n, dg, ci // dg, h * w)
    y0, x0 = torch.floor(y), torch.floor(x)
    fy, fx = y - y0, x - x0
    v = ((1 - fy) * (1 - fx) * _corner(img, y0, x0, h, w) + (1 - fy) * fx * _corner(img, y0, x0 + 1, h, w)
         + fy * (1 - fx) * _corner(img, y0 + 1, x0, h, w) + fy * fx * _corner(img, y0 + 1, x0 + 1, h, w))
    if s["mk"] is not None:
        v = v * s["mk"].to(real).reshape(n, dg, 1, -1)
    return v.reshape(n, ci, k * k, ho * wo)


def _plain_deform(s):
    n, gr, o = s["n"], s["groups"], s["out"]
    col = _columns(s, torch.float32).reshape(n, gr, -1, _out_size(s)[0] * _out_size(s)[1]).mT
    q, scale = _codes(col)
    w = s["wq"].contiguous().float().view(1, gr, o // gr, -1)
    y = (w @ q.mT) * scale.mT * s["ws"].view(1, gr, -1, 1)
    y = y.reshape(n, o, *_out_size(s))
    return (y if s["b"] is None else y + s["b"].float()[:, None, None]).to(_out_type(s))


def _out_type(s):
    """float32 images are answered in bf16, as the layers behind an 8-bit one take them."""
    return torch.bfloat16 if s["dtype"] == "float32" else _DTYPES[s["dtype"]]


# ---- the package's operators ---------------------------------------------------


def _own(s):
    import pytorch_mps_deform_conv2d_b200 as dcn

    if s["op"] == "ns":
        return dcn.newton_schulz(s["x"], steps=5, coefficients=(A, B, C), eps=EPS)
    if s["op"] == "muon":
        dcn.muon_update_(s["p"], s["g"], s["m"], lr=LR, momentum=MOMENTUM, nesterov=s["nesterov"], weight_decay=DECAY, steps=5,
                         coefficients=(A, B, C), eps=EPS)
        return {"p": s["p"], "m": s["m"]}
    if s["op"] == "linear":
        return dcn.int8_linear(s["x"], s["wq"], s["ws"], s["b"], x_scale=s["xs"], out_dtype=_DTYPES[s["dtype"]])
    return dcn.deform_conv2d_int8(s["x"], s["off"], s["wq"], s["ws"], s["b"], stride=s["s"], padding=s["p"], dilation=s["d"], mask=s["mk"],
                                  out_dtype=_out_type(s))


def run(state):
    if own:
        return _own(state)
    if state["op"] == "ns":
        return _orthogonal(state["x"]).to(state["x"].dtype)
    if state["op"] == "muon":
        return _plain_muon(state)
    return _plain_linear(state) if state["op"] == "linear" else _plain_deform(state)


# ---- what a pass needs, and the exact answers ----------------------------------


def _quintic_flops(rows, cols):
    """Five steps on a matrix; the two symmetric products count half."""
    m, n = min(rows, cols), max(rows, cols)
    return 5.0 * (m * m * n + m * m * m + 2 * m * m * n)


def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "ns":
        n = case["batch"] * case["rows"] * case["cols"]
        return {"bytes": 2 * e * n, "flops": case["batch"] * _quintic_flops(case["rows"], case["cols"])}
    if case["op"] == "muon":
        rows, cols = case["out"], case["cin"] * case["k"] ** 2
        # gradient read, parameter and float32 momentum read and written
        return {"bytes": case["layers"] * rows * cols * (3 * e + 8), "flops": case["layers"] * _quintic_flops(rows, cols)}
    if case["op"] == "linear":
        m, n, k = case["tokens"], case["out"], case["cin"]
        return {"bytes": m * k * (1 if case["given"] else e) + n * k + m * n * e + 4 * n, "flops": 2.0 * m * n * k}
    ho, wo = _out_size(case)
    pixels, kk = case["n"] * ho * wo, case["k"] ** 2
    samples = pixels * kk * case["cin"]
    per_tap = 3 if case["mask"] else 2
    return {"bytes": e * (case["n"] * case["cin"] * case["h"] * case["w"] + pixels * per_tap * case["dg"] * kk) + 2 * pixels * case["out"]
            + case["out"] * case["cin"] // case["groups"] * kk,
            "flops": 2.0 * samples * case["out"] / case["groups"] + 8.0 * samples}


def _exact_orthogonal(u):
    """Five steps by the singular values' side: X = P(U U^T) U, each from the recurrence in 64 bits."""
    x = u / (torch.linalg.matrix_norm(u, keepdim=True) + EPS)
    flip = x.shape[-2] > x.shape[-1]
    x = x.transpose(-2, -1) if flip else x
    eye = torch.eye(x.shape[-2], dtype=torch.float64, device=x.device)
    for _ in range(5):
        s = torch.matmul(x, x.transpose(-2, -1))
        x = torch.matmul(A * eye + torch.matmul(s, B * eye + C * s), x)
    return x.transpose(-2, -1) if flip else x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "ns":
        return _exact_orthogonal(s["x"].double())
    if case["op"] == "muon":
        shrink = max(1.0, case["out"] / (case["cin"] * case["k"] ** 2)) ** 0.5
        ps, ms = [], []
        for p, g, m in zip(s["p"], s["g"], s["m"]):
            g, m = g.double(), m.double()
            m = m + (1 - MOMENTUM) * (g - m)
            u = g + MOMENTUM * (m - g) if case["nesterov"] else m
            ps.append(p.double() * (1 - LR * DECAY) - LR * shrink * _exact_orthogonal(u.flatten(1)).reshape(p.shape))
            ms.append(m)
        return {"p": ps, "m": ms}
    if case["op"] == "linear":
        if case["given"]:
            q, scale = s["x"].double(), s["xs"].double()
        else:
            x = s["x"].double()
            scale = x.abs().max(1).values / 127
            q = torch.round(x / scale.clamp(min=1e-300)[:, None])
        y = torch.einsum("mk,nk->mn", q, s["wq"].double()) * torch.outer(scale, s["ws"].double())
        return y if s["b"] is None else y + s["b"].double()
    # by bilinear hats: a pixel (i, j) counts max(0, 1 - |y - i|) max(0, 1 - |x - j|)
    n, gr, o, k, dg = case["n"], case["groups"], case["out"], case["k"], case["dg"]
    ho, wo = _out_size(case)
    off = s["off"].double().reshape(n, dg, k * k, 2, ho, wo)
    wq = s["wq"].double().reshape(gr, o // gr, -1)
    out = torch.empty(n, o, ho * wo, dtype=torch.float64, device="cuda")
    ys, xs = torch.meshgrid(torch.arange(ho, device="cuda"), torch.arange(wo, device="cuda"), indexing="ij")
    for b in range(n):
        col = torch.empty(dg, case["cin"] // dg, k * k, ho * wo, dtype=torch.float64, device="cuda")
        pad = torch.nn.functional.pad(s["x"][b].double(), (1, 1, 1, 1)).reshape(dg, case["cin"] // dg, -1)
        for t in range(k * k):
            y = ys * case["s"] - case["p"] + (t // k) * case["d"] + off[b, :, t, 0]
            x = xs * case["s"] - case["p"] + (t % k) * case["d"] + off[b, :, t, 1]
            v = 0.0
            for dy in (0, 1):
                for dx in (0, 1):
                    i, j = torch.floor(y) + dy, torch.floor(x) + dx
                    hat = torch.relu(1 - (y - i).abs()) * torch.relu(1 - (x - j).abs())
                    at = (i.clamp(-1, case["h"]) + 1) * (case["w"] + 2) + j.clamp(-1, case["w"]) + 1  # the padded border holds zeros
                    v = v + hat.reshape(dg, 1, -1) * torch.take_along_dim(pad, at.long().reshape(dg, 1, -1), 2)
            col[:, :, t] = v if s["mk"] is None else v * s["mk"][b].double().reshape(dg, k * k, 1, -1)[:, t]
        col = col.reshape(gr, -1, ho * wo)
        scale = col.abs().max(1, keepdim=True).values / 127
        q = torch.round(col / scale.clamp(min=1e-300))
        out[b] = (torch.matmul(wq, q) * scale * s["ws"].double().reshape(gr, -1, 1)).reshape(o, -1)
    out = out.reshape(n, o, ho, wo)
    return out if s["b"] is None else out + s["b"].double()[:, None, None]
