"""The norms around a block with its gate and residual scale (nn.GatedResidualNorm, fbfc_residual_norm_*): against the
formulas in 64 bits, their gradients by automatic differentiation there, and against differences."""
import ctypes

import pytest
import torch

from fbcunn_amd import _lib

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
FORMS = {"full": (1, 1, 1), "ungated": (1, 0, 1), "last": (1, 1, 0), "first": (0, 0, 1), "ungated last": (1, 0, 0)}
EPS = 1e-6


# refusals: no GPU needed ------------------------------------------------------------------------------

P = 0x1000


def _rows(data=P, stride=8):
    return ctypes.byref(_lib.Rows(data, stride))


def _forward(rows=2, channels=8, type=0, eps=1e-6, **kw):
    d = _lib.ResidualNormDesc(rows, channels, type, eps)
    a = dict(residual=_rows(), branch=_rows(), gate=_rows(), post=P, scale=P, pre=P, output=_rows(), normed=_rows())
    a.update(kw)
    rc = _lib.lib().fbfc_residual_norm_forward(ctypes.byref(d), *a.values(), None)
    return rc, _lib.lib().fbfc_last_error().decode()


def _backward(rows=2, channels=8, type=0, eps=1e-6, **kw):
    d = _lib.ResidualNormDesc(rows, channels, type, eps)
    a = dict(residual=_rows(), branch=_rows(), gate=_rows(), post=P, scale=P, pre=P, gr=_rows(), gn=_rows(), dr=_rows(),
             dy=_rows(), dz=_rows(), dpost=P, dscale=P, dpre=P, factor=1.0, workspace=P)
    a.update(kw)
    rc = _lib.lib().fbfc_residual_norm_backward(ctypes.byref(d), *a.values(), None)
    return rc, _lib.lib().fbfc_last_error().decode()


@pytest.mark.parametrize("call", [_forward, _backward])
@pytest.mark.parametrize("kw,text", [
    (dict(rows=-1), "positive"), (dict(channels=0), "positive"), (dict(type=3), "type"), (dict(eps=0.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(residual=None), "residual"), (dict(branch=None), ""), (dict(post=None), "weight"),
    (dict(scale=None), "scale"), (dict(pre=None), "weight"), (dict(residual=_rows(0x1002)), "aligned"),
    (dict(gate=_rows(P, -8)), "overlap"), (dict(branch=_rows(0)), ""),
])
def test_refusals(call, kw, text):
    rc, message = call(**kw)
    assert rc == _lib.ERR_INVALID_ARGUMENT and text in message, message


def test_more_refusals():
    assert _forward(channels=16385)[0] == _lib.ERR_UNSUPPORTED_SIZE
    assert _lib.lib().fbfc_residual_norm_forward(None, *([None] * 9)) == _lib.ERR_INVALID_ARGUMENT
    for kw, text in ((dict(output=None, normed=None, branch=None, gate=None), "nothing"), (dict(output=None), "branch"),
                     (dict(output=_rows(P, 7)), "overlap"), (dict(normed=_rows(0x1001)), "aligned")):
        rc, message = _forward(**kw)
        assert rc == _lib.ERR_INVALID_ARGUMENT and text in message, (kw, message)
    for kw, text in ((dict(gr=None, gn=None), "gradient"), (dict(gate=None), "gate"), (dict(workspace=None), "workspace"),
                     (dict(branch=None, gate=None, dz=None), "branch"), (dict(dr=_rows(P, 7)), "overlap"),
                     (dict(gn=_rows(0x1001)), "aligned")):
        rc, message = _backward(**kw)
        assert rc == _lib.ERR_INVALID_ARGUMENT and text in message, (kw, message)
    assert _forward(rows=0)[0] == _lib.OK
    d = _lib.ResidualNormDesc(0, 8, 0, 1e-6)
    assert _lib.lib().fbfc_residual_norm_workspace_bytes(ctypes.byref(d)) == 0


def test_module_refusals_without_gpu():
    from fbcunn_amd import nn
    with pytest.raises(ValueError):
        nn.GatedResidualNorm(0, device="cpu")
    with pytest.raises(ValueError):
        nn.GatedResidualNorm(8, branch=False, norm=False, device="cpu")
    with pytest.raises(TypeError):
        nn.GatedResidualNorm(8, device="cpu").updateOutput([torch.zeros(2, 8)] * 3)


# plain forms ---------------------------------------------------------------------------------------------

def _net(channels, form, seed):
    from fbcunn_amd import nn
    b, g, n = FORMS[form]
    net = nn.GatedResidualNorm(channels, eps=EPS, branch=bool(b), gate=bool(g), norm=bool(n))
    gen = torch.Generator("cuda").manual_seed(seed)
    for p, mean in zip(net.parameters()[0], (1.0, 0.5, 1.0) if b else (1.0,)):
        p.copy_(mean + 0.2 * torch.randn(channels, generator=gen, device="cuda"))
    return net


def _inputs(shape, form, dtype, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    b, g, n = FORMS[form]
    make = lambda s: (torch.randn(*shape, generator=gen, device="cuda") * s).to(dtype)   # noqa: E731
    inputs = [make(2.0)] + ([make(0.7)] if b else []) + ([make(1.5)] if g else [])
    return inputs, [make(1.0), make(1.0) if n else None]


def _plain(net, inputs, grads=None, factor=1.0):
    """Values and bounds in 64 bits: {name: (value, bound of the error before the last rounding)}."""
    leaf = lambda t: None if t is None else t.detach().cpu().double().requires_grad_(True)   # noqa: E731
    r0 = leaf(inputs[0])
    y = leaf(inputs[1]) if net.hasBranch else None
    z = leaf(inputs[2]) if net.hasGate else None
    post, scale, pre = leaf(net.postWeight), leaf(net.scale), leaf(net.preWeight)
    out, size, u = r0, r0.detach().abs(), None
    if y is not None:
        i1 = (y.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
        yn = y * i1
        k = torch.sigmoid(z) if z is not None else torch.ones_like(y)
        u = yn * post * scale
        out = r0 + k * u
        size = size + (k * u).detach().abs()
    # Sums of squares: 16 terms in a lane, six steps over the lanes, 16 wavefronts, half of that for the root; the
    # exponential of z is off by |z| + 2 units and |z| < 10 here: 64 units cover a forward value
    res = {"output": (out.detach(), 64 * U * size)}
    n = None
    if pre is not None:
        i2 = (out.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
        n = out * i2 * pre
        res["normed"] = (n.detach(), 64 * U * (size * i2 * pre.abs() + n.abs()).detach())
    if grads is None:
        return res
    gr, gn = (None if g is None else g.detach().cpu().double() for g in grads)
    loss = 0
    if gr is not None:
        loss = loss + (out * gr).sum()
    if gn is not None:
        loss = loss + (n * gn).sum()
    loss.backward()
    with torch.no_grad():
        # the same sums of magnitudes; each further stage of products and sums adds units
        a = torch.zeros_like(r0) if gr is None else gr.abs()
        if gn is not None:
            w, rn = (gn * pre).abs(), size * i2
            a = a + i2 * (w + rn * (w * rn).mean(-1, keepdim=True))
            res["gradPreWeight"] = (pre.grad * factor, 512 * U * abs(factor) * (gn.abs() * rn).flatten(0, -2).sum(0))
        elif pre is not None:
            res["gradPreWeight"] = (torch.zeros_like(pre), torch.zeros_like(pre))
        res["gradInput0"] = (r0.grad, 128 * U * a)
        if y is not None:
            b = a * k * (post * scale).abs()
            res["gradInput1"] = (y.grad, 256 * U * i1 * (b + yn.abs() * (b * yn.abs()).mean(-1, keepdim=True)))
            q = (a * k * yn.abs()).flatten(0, -2).sum(0)
            res["gradPostWeight"] = (post.grad * factor, 512 * U * abs(factor) * q * scale.abs())
            res["gradScale"] = (scale.grad * factor, 512 * U * abs(factor) * q * post.abs())
        if z is not None:
            res["gradInput2"] = (z.grad, 256 * U * a * u.abs() * k * (1 - k))
    return res


def _check(got, want, what):
    value, bound = want
    x = got.detach().cpu().double()
    tol = bound + 1e-37
    if got.dtype != torch.float32:
        tol = tol + torch.finfo(got.dtype).eps / 2 * (value.abs() + bound) + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    else:
        tol = tol + U * value.abs()
    off = (x - value).abs()
    assert bool((off <= tol).all()), "%s: %g times the bound" % (what, float((off / tol).max()))


def _check_all(net, inputs, grads, factor=1.0):
    want = _plain(net, inputs, grads, factor)
    output, normed = net.updateOutput(inputs)
    if not net.hasBranch:
        assert output is inputs[0]
    net.backward(inputs, grads, factor)
    got = {"output": output, "normed": normed, "gradPostWeight": net.gradPostWeight, "gradScale": net.gradScale,
           "gradPreWeight": net.gradPreWeight}
    got.update({"gradInput%d" % i: t for i, t in enumerate(net.gradInput)})
    for name, w in want.items():
        _check(got[name], w, name)
    return got


# rows x channels: around every change of the number of lanes and of vectors, rows few and many
SHAPES = [(1, 1), (5, 3), (2, 8), (33, 63), (70, 64), (9, 65), (300, 130), (3, 255), (1, 512), (700, 513), (1300, 257),
          (1, 1000), (601, 1000), (2, 2048), (513, 2050), (3, 4096), (700, 1025), (515, 4100), (2, 8192), (600, 5001), (3, 8193),
          (530, 8200), (2, 16384), (520, 12001)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % s)
def test_values_and_gradients(shape, dtype):
    net = _net(shape[1], "full", 1)
    inputs, grads = _inputs(shape, "full", TYPES[dtype], shape[0] + shape[1])
    _check_all(net, inputs, grads, 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", [f for f in FORMS if f != "full"])
@pytest.mark.parametrize("shape", [(7, 40), (30, 300), (600, 1100)], ids=lambda s: "%dx%d" % s)
def test_forms(shape, form, dtype):
    net = _net(shape[1], form, 2)
    inputs, grads = _inputs(shape, form, TYPES[dtype], 3)
    _check_all(net, inputs, grads)
    if grads[1] is not None:       # either gradient alone
        _check_all(net, inputs, [None, grads[1]])
        _check_all(net, inputs, [grads[0], None])


@pytest.mark.gpu
def test_many_rows_are_walked_over():
    """More rows than workgroups, narrow and wide: rows beyond the first round and their part of the sums."""
    for shape in ((40000, 24), (9000, 200), (5000, 1025)):
        net = _net(shape[1], "full", 1)
        inputs, grads = _inputs(shape, "full", torch.bfloat16, 5)
        _check_all(net, inputs, grads)


@pytest.mark.gpu
def test_halves_match_the_whole_and_calls_repeat():
    net = _net(1000, "full", 1)
    inputs, grads = _inputs((77, 1000), "full", torch.bfloat16, 5)
    net.backward(inputs, grads, 2.0)
    first = [t.clone() for t in net.gradInput + net.parameters()[1]]
    for t in net.gradInput + net.parameters()[1]:
        t.fill_(float("nan"))
    net.updateGradInput(inputs, grads)
    assert all(t.isnan().all() for t in net.parameters()[1])
    net.accGradParameters(inputs, grads, 2.0)
    for a, b in zip(first, net.gradInput + net.parameters()[1]):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("channels", [37, 777, 9000])
def test_rows_of_a_wider_storage(channels):
    """Strided rows at odd addresses, one broadcast over the rows; what lies beside what is written stays."""
    L = _lib.lib()
    rows, dtype = 11, torch.bfloat16
    net = _net(channels, "full", 1)
    inputs, grads = _inputs((rows, channels), "full", dtype, 5)
    inputs[2] = inputs[2][:1].expand(rows, channels)
    wide = torch.full((10, rows, channels + 5), 7.0, dtype=dtype, device="cuda")
    views = [w.view(-1)[1 + i:1 + i + rows * (channels + 3)].view(rows, channels + 3)[:, :channels] for i, w in enumerate(wide)]
    given = []
    for v, t in zip(views[:4], [inputs[0], inputs[1], grads[0], grads[1]]):
        v.copy_(t)
        given.append(v)
    r = lambda t: ctypes.byref(_lib.Rows(t.data_ptr(), t.stride(0)))   # noqa: E731
    p = lambda t: t.data_ptr()   # noqa: E731
    d = ctypes.byref(_lib.ResidualNormDesc(rows, channels, _lib.BF16, EPS))
    gate = inputs[2]
    outs = views[4:9]
    st = torch.cuda.current_stream().cuda_stream
    _lib.check(L.fbfc_residual_norm_forward(d, r(given[0]), r(given[1]), r(gate), p(net.postWeight), p(net.scale), p(net.preWeight),
                                            r(outs[0]), r(outs[1]), st))
    ws = torch.empty(L.fbfc_residual_norm_workspace_bytes(d), dtype=torch.uint8, device="cuda")
    _lib.check(L.fbfc_residual_norm_backward(d, r(given[0]), r(given[1]), r(gate), p(net.postWeight), p(net.scale), p(net.preWeight),
                                             r(given[2]), r(given[3]), r(outs[2]), r(outs[3]), r(outs[4]), p(net.gradPostWeight),
                                             p(net.gradScale), p(net.gradPreWeight), 1.0, p(ws), st))
    want = _plain(net, [inputs[0], inputs[1], gate.contiguous()], grads)
    for name, t in zip(("output", "normed", "gradInput0", "gradInput1", "gradInput2"), outs):
        _check(t, want[name], name)
    for name in ("gradPostWeight", "gradScale", "gradPreWeight"):
        _check(getattr(net, name), want[name], name)
    for v, w in zip(views, wide):
        v.fill_(7.0)
        assert bool((w == 7).all())


@pytest.mark.gpu
def test_outputs_in_the_place_of_inputs():
    L = _lib.lib()
    net = _net(600, "full", 1)
    inputs, _ = _inputs((50, 600), "full", torch.float32, 5)
    want = [t.clone() for t in net.updateOutput(inputs)]
    r = lambda t: ctypes.byref(_lib.Rows(t.data_ptr(), 600))   # noqa: E731
    p = lambda t: t.data_ptr()   # noqa: E731
    d = ctypes.byref(_lib.ResidualNormDesc(50, 600, _lib.F32, EPS))
    _lib.check(L.fbfc_residual_norm_forward(d, r(inputs[0]), r(inputs[1]), r(inputs[2]), p(net.postWeight), p(net.scale),
                                            p(net.preWeight), r(inputs[0]), r(inputs[1]), torch.cuda.current_stream().cuda_stream))
    assert torch.equal(inputs[0], want[0]) and torch.equal(inputs[1], want[1])


@pytest.mark.gpu
def test_special_rows():
    """A row of zeros has finite results; one with a NaN or an infinity leaves the others as they are."""
    for channels in (40, 700):
        net = _net(channels, "full", 1)
        inputs, grads = _inputs((6, channels), "full", torch.float32, 5)
        for t in inputs[:2]:
            t[1] = 0
        inputs[2][1, 0], inputs[2][1, 1], inputs[2][1, 2] = float("inf"), -float("inf"), -200.0   # gates fully open and closed
        want = [t.clone() for t in net.updateOutput(inputs)] + [t.clone() for t in net.backward(inputs, grads)]
        assert all(bool(t.isfinite().all()) for t in want)
        _check_all(net, [inputs[0], inputs[1], inputs[2].clamp(-200, 200)], grads)
        inputs[1][3, 7], inputs[0][5, 9] = float("nan"), float("inf")
        got = net.updateOutput(inputs) + net.backward(inputs, grads)
        keep = [0, 1, 2, 4]
        for a, b in zip(want, got):
            assert torch.equal(a[keep], b[keep])
        assert bool(got[1][3].isnan().all()) and not bool(got[1][5].isfinite().all())


@pytest.mark.gpu
def test_gradient_against_differences():
    """Directional derivative of the forward pass by central differences.  Bounds: the rounding of the forward pass over
    the step, and how far the same difference in 64 bits is from the gradient in 64 bits."""
    rows, channels, h = 4, 24, 2.0 ** -6
    net = _net(channels, "full", 1)
    inputs, grads = _inputs((rows, channels), "full", torch.float32, 5)
    moves, _ = _inputs((rows, channels), "full", torch.float32, 6)
    net.backward(inputs, grads)
    mine = sum(float((g.double() * m.double()).sum()) for g, m in zip(net.gradInput, moves))
    want = _plain(net, inputs, grads)
    exact = sum(float((want["gradInput%d" % i][0] * m.cpu().double()).sum()) for i, m in enumerate(moves))
    sums, plain, rounding = [], [], 0.0
    for sign in (1, -1):
        at = [t + sign * h * m for t, m in zip(inputs, moves)]
        out, ref = net.updateOutput(at), _plain(net, at)
        sums.append(sum(float((o.double() * g.double()).sum()) for o, g in zip(out, grads)))
        plain.append(sum(float((ref[k][0] * g.cpu().double()).sum()) for k, g in zip(("output", "normed"), grads)))
        rounding += sum(float(((ref[k][1] + U * ref[k][0].abs()) * g.cpu().double().abs()).sum()) for k, g in zip(("output", "normed"), grads))
    tol = rounding / (2 * h) + 1.01 * abs((plain[0] - plain[1]) / (2 * h) - exact) + 256 * U * sum(float((want["gradInput%d" % i][1] / U * m.cpu().abs()).sum()) for i, m in enumerate(moves)) / 256
    assert abs((sums[0] - sums[1]) / (2 * h) - mine) <= tol
    assert tol < 0.05 * abs(exact)


@pytest.mark.gpu
def test_replays_from_a_graph():
    net = _net(1000, "full", 1)
    inputs, grads = _inputs((70, 1000), "full", torch.bfloat16, 5)

    def step():
        net.updateOutput(inputs)
        net.backward(inputs, grads)

    results = lambda: net.output + net.gradInput + net.parameters()[1]   # noqa: E731
    step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    other, more = _inputs((900, 1000), "full", torch.bfloat16, 6)
    big = _net(1000, "full", 1)
    for rep in range(3):
        inputs[0].mul_(-0.5)
        for t in results():
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in results()]
        big.updateOutput(inputs), big.backward(inputs, grads)
        for a, b in zip(got, big.output + big.gradInput + big.parameters()[1]):
            assert torch.equal(a, b), rep
        net._workspace.take(1 << 22, inputs[0].device)     # outgrown workspaces stay for the graph
        (inputs[0].float() * 2).sum().item()


@pytest.mark.gpu
def test_module_refusals_and_shapes():
    net = _net(16, "full", 1)
    x = torch.randn(2, 3, 16, device="cuda")
    out, normed = net.updateOutput([x, x * 0.5, x])
    assert out.shape == normed.shape == x.shape
    assert [tuple(t.shape) for t in net.backward([x, x, x], [x, x])] == [(2, 3, 16)] * 3
    empty = x[:0]
    assert net.updateOutput([empty, empty, empty])[0].shape == (0, 3, 16)
    net.backward([empty, empty, empty], [empty, empty])
    assert all(bool((g == 0).all()) for g in net.parameters()[1])
    for bad, error in (([x, x], ValueError), ([x, x, x[:1]], ValueError), ([x, x, x.half()], TypeError),
                       ([x.double()] * 3, TypeError), ([x[..., :8]] * 3, ValueError), ([x.cpu()] * 3, TypeError),
                       ([x.transpose(0, 1)] * 3, ValueError), ([torch.randn(3, 32, device="cuda")[:, ::2]] * 3, ValueError)):
        with pytest.raises(error):
            net.updateOutput(bad)
    with pytest.raises(ValueError):
        net.backward([x, x, x], [None, None])
    with pytest.raises(ValueError):
        _net(16, "last", 1).backward([x, x, x], [x, x])
    with pytest.raises(_lib.FbfcError):
        _net(16385, "first", 1).updateOutput([torch.zeros(2, 16385, device="cuda")])


def test_misaligned_weights_are_refused():
    for kw in (dict(post=0x1002), dict(scale=0x1001), dict(pre=0x1002)):
        for call in (_forward, _backward):
            rc, message = call(**kw)
            assert rc == _lib.ERR_INVALID_ARGUMENT and "4 bytes" in message
    for kw in (dict(dpost=0x1002), dict(dscale=0x1002), dict(dpre=0x1002)):
        assert _backward(**kw)[0] == _lib.ERR_INVALID_ARGUMENT


@pytest.mark.gpu
def test_own_output_as_residual_and_a_changed_eps():
    """The next block's residual is this module's output: it keeps its values.  eps is read at each call."""
    net = _net(48, "full", 1)
    inputs, grads = _inputs((6, 48), "full", torch.float32, 5)
    first = net.updateOutput(inputs)
    kept = [t.clone() for t in first]
    again = net.updateOutput([first[0], inputs[1], inputs[2]])
    assert again[0] is not first[0] and torch.equal(first[0], kept[0])
    _check(again[1], _plain(net, [kept[0], inputs[1], inputs[2]])["normed"], "normed")
    wide = net.updateOutput(inputs)[1].clone()
    net.eps = 1.0
    assert not torch.equal(net.updateOutput(inputs)[1], wide)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """2.3 thousand million elements: the last rows as a tensor of their own, forward and backward."""
    rows, channels = 140000, 16384
    net, part = _net(channels, "ungated", 1), _net(channels, "ungated", 1)
    gen = torch.Generator("cuda").manual_seed(2)
    x, y = (torch.empty(rows, channels, dtype=torch.bfloat16, device="cuda").normal_(generator=gen) for _ in range(2))
    net.updateOutput([x, y])
    tail = [x[-64:], y[-64:]]
    for a, b in zip(net.output, part.updateOutput(tail)):
        assert torch.equal(a[-64:], b)
    net.updateGradInput([x, y], [x, y])
    for a, b in zip(net.gradInput, part.updateGradInput(tail, tail)):
        assert torch.equal(a[-64:], b)


@pytest.mark.gpu
def test_parameters_on_another_device_are_refused():
    from fbcunn_amd import nn
    x = torch.randn(2, 16, device="cuda")
    with pytest.raises(ValueError, match="another device"):
        nn.GatedResidualNorm(16, device="cpu").updateOutput([x, x, x])


@pytest.mark.gpu
def test_a_view_of_the_own_output_as_residual_keeps_its_values():
    net = _net(48, "full", 1)
    inputs, _ = _inputs((6, 48), "full", torch.float32, 6)
    first = net.updateOutput(inputs)[0]
    kept = first.clone()
    again = net.updateOutput([first.view(6, 48), inputs[1], inputs[2]])
    assert again[0] is not first and torch.equal(first, kept)
    _check(again[1], _plain(net, [kept, inputs[1], inputs[2]])["normed"], "normed")


@pytest.mark.gpu
def test_a_graph_keeps_its_results_when_the_module_goes_on_with_other_shapes():
    net, other = _net(40, "full", 1), _net(40, "full", 1)
    inputs, grads = _inputs((70, 40), "full", torch.float32, 7)

    def step(m, n=70):
        m.updateOutput([t[:n] for t in inputs])
        m.backward([t[:n] for t in inputs], [t[:n] for t in grads])

    step(net)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(net)
    out, normed = net.output
    for n in (30, 70, 1):
        step(net, n)
    fill = [torch.full((70 * 40,), 7.0, device="cuda") for _ in range(20)]   # memory that the module has given back would be found here
    for rep in range(3):
        inputs[0].mul_(-0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(bool((t == 7.0).all()) for t in fill)
        step(other)
        assert torch.equal(out, other.output[0]) and torch.equal(normed, other.output[1])
        assert torch.equal(net.gradScale, other.gradScale)


@pytest.mark.gpu
def test_own_gradients_as_inputs_keep_their_values():
    """What the module's last call gave is an input of the next, whose halves both have to find it as it was."""
    net, other = _net(48, "full", 1), _net(48, "full", 1)
    inputs, grads = _inputs((6, 48), "full", torch.float32, 8)

    def halves(m, inputs, grads):
        m.updateOutput(inputs)
        m.updateGradInput(inputs, grads)
        m.accGradParameters(inputs, grads)

    halves(net, inputs, grads)
    for i in range(3):
        for place in range(5):
            mine = net.gradInput[i]
            kept = mine.clone()
            given = [(inputs + grads)[:place] + [t] + (inputs + grads)[place + 1:] for t in (mine, kept)]
            halves(net, given[0][:3], given[0][3:])
            halves(other, given[1][:3], given[1][3:])
            assert torch.equal(mine, kept), (i, place)
            for a, b in zip(net.output + net.gradInput + net.parameters()[1], other.output + other.gradInput + other.parameters()[1]):
                assert torch.equal(a, b), (i, place)


@pytest.mark.gpu
def test_parameters_that_do_not_fit_are_refused():
    net = _net(48, "full", 1)
    inputs, grads = _inputs((6, 48), "full", torch.float32, 9)
    net.updateOutput(inputs)
    net.backward(inputs, grads)
    for name in ("postWeight", "scale", "preWeight", "gradPostWeight", "gradScale", "gradPreWeight"):
        whole = getattr(net, name)
        for bad, error in ((whole.half(), TypeError), (whole[:47], ValueError), (whole.cpu(), ValueError), (list(whole), TypeError)):
            setattr(net, name, bad)
            with pytest.raises(error, match=name):
                net.backward(inputs, grads)
            with pytest.raises(error, match=name):
                net.accGradParameters(inputs, grads)
            if not name.startswith("grad"):
                with pytest.raises(error, match=name):
                    net.updateOutput(inputs)
        setattr(net, name, whole)
    net.updateOutput(inputs)
    net.backward(inputs, grads)


@pytest.mark.gpu
def test_a_module_works_on_after_its_buffers_are_cleaned_up():
    net = _net(40, "full", 1)
    inputs, grads = _inputs((70, 40), "full", torch.float32, 10)
    want = [t.clone() for t in net.updateOutput(inputs) + net.backward(inputs, grads) + net.parameters()[1]]
    assert len(net._workspace._of) == 1
    net.cleanupBuffers()
    assert not net._workspace._of
    for t in net.parameters()[1]:
        t.fill_(float("nan"))
    for a, b in zip(want, net.updateOutput(inputs) + net.backward(inputs, grads) + net.parameters()[1]):
        assert torch.equal(a, b)
