"""The gated linear recurrence (nn.GatedLinearRecurrence, fbfc_recurrence_*): values and gradients against one step after
the other in 64 bits, with bounds that are carried through the same recurrence."""
import ctypes

import pytest
import torch

from fbcunn_amd import _lib

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# refusals: no GPU needed ------------------------------------------------------------------------------

P = 0x1000


def _st(data=P, sb=80, st=8, sc=1):
    return ctypes.byref(_lib.Steps(data, sb, st, sc))


def _forward(batch=2, channels=8, steps=10, type=0, **kw):
    d = _lib.RecurrenceDesc(batch, channels, steps, type)
    a = dict(x=_st(), gate=_st(), bias=None, state_in=None, lengths=None, y=_st(), state_out=P, checkpoints=None, workspace=P)
    a.update(kw)
    rc = _lib.lib().fbfc_recurrence_forward(ctypes.byref(d), *a.values(), None)
    return rc, _lib.lib().fbfc_last_error().decode()


def _backward(batch=2, channels=8, steps=10, type=0, **kw):
    d = _lib.RecurrenceDesc(batch, channels, steps, type)
    a = dict(x=_st(), gate=_st(), bias=None, lengths=None, checkpoints=P, y=_st(), gstate=None, gx=_st(), gz=_st(), gb=P, factor=1.0,
             gstate_in=P, workspace=P)
    a.update(kw)
    rc = _lib.lib().fbfc_recurrence_backward(ctypes.byref(d), *a.values(), None)
    return rc, _lib.lib().fbfc_last_error().decode()


@pytest.mark.parametrize("call", [_forward, _backward])
@pytest.mark.parametrize("kw,text", [
    (dict(batch=-1), "positive"), (dict(channels=0), "positive"), (dict(steps=-1), "positive"), (dict(type=7), "type"),
    (dict(x=None), "needed"), (dict(gate=_st(0)), "needed"), (dict(y=None), "needed"), (dict(x=_st(0x1002)), "aligned"),
    (dict(workspace=None), "workspace"), (dict(workspace=0x1008), "workspace"),
])
def test_refusals(call, kw, text):
    rc, message = call(**kw)
    assert rc == _lib.ERR_INVALID_ARGUMENT and text in message, message


def test_more_refusals():
    for bad in (_st(sb=79), _st(st=7), _st(sc=0), _st(sb=-80), _st(sb=8, st=8), _st(sb=80, st=1, sc=9)):
        rc, message = _forward(y=bad)
        assert rc == _lib.ERR_INVALID_ARGUMENT and "overlap" in message
        for k in ("gx", "gz"):
            rc, message = _backward(**{k: bad})
            assert rc == _lib.ERR_INVALID_ARGUMENT and "overlap" in message
    rc, message = _backward(checkpoints=None)
    assert rc == _lib.ERR_INVALID_ARGUMENT and "checkpoints" in message
    assert _forward(batch=1 << 30, channels=1 << 30)[0] == _lib.ERR_UNSUPPORTED_SIZE
    assert _forward(batch=1 << 20, channels=1 << 17, steps=1 << 39)[0] == _lib.ERR_UNSUPPORTED_SIZE
    L = _lib.lib()
    assert L.fbfc_recurrence_forward(None, *([None] * 10)) == _lib.ERR_INVALID_ARGUMENT
    assert L.fbfc_recurrence_checkpoint_bytes(None) == 0 and L.fbfc_recurrence_workspace_bytes(None) == 0
    assert _forward(batch=0)[0] == _lib.OK


def test_checkpoints_are_small():
    d = _lib.RecurrenceDesc(3, 100, 1000, _lib.BF16)
    assert _lib.lib().fbfc_recurrence_checkpoint_bytes(ctypes.byref(d)) == 3 * 100 * 8 * 4


def test_module_refusals_without_gpu():
    from fbcunn_amd import nn
    with pytest.raises(ValueError):
        nn.GatedLinearRecurrence(0, device="cpu")
    with pytest.raises(TypeError):
        nn.GatedLinearRecurrence(8, device="cpu").updateOutput([torch.zeros(2, 3, 8)] * 2)


# plain form ----------------------------------------------------------------------------------------------

def _plain(x, gate, bias, h0=None, lengths=None, gy=None, gh=None, factor=1.0):
    """{name: (value, bound before the last rounding)}, one step after the other in 64 bits.  The bounds count, for gates
    below 10: 24 units of 1 - a (its exponential is off by |z| + 2), 10 of a, 2 of each sum."""
    up = lambda t: None if t is None else t.detach().cpu().double()   # noqa: E731
    x, gate, bias, gy, gh = up(x), up(gate), up(bias), up(gy), up(gh)
    B, T, D = x.shape
    n = torch.full((B,), T) if lengths is None else lengths.cpu().clamp(0, T)
    z = gate + bias
    a, c = torch.sigmoid(z), torch.sigmoid(-z)
    live = torch.arange(T)[None, :, None] < n[:, None, None]
    x, a, c = torch.where(live, x, 0.0), torch.where(live, a, 1.0), torch.where(live, c, 0.0)
    h = torch.zeros(B, D, dtype=torch.float64) if h0 is None else up(h0).clone()
    e = torch.zeros_like(h)
    H, E, before, Eb = (torch.zeros(B, T, D, dtype=torch.float64) for _ in range(4))
    for t in range(T):
        before[:, t], Eb[:, t] = h, e
        new = a[:, t] * h + c[:, t] * x[:, t]
        e = a[:, t] * e + U * (24 * c[:, t] * (x[:, t].abs() + h.abs()) + 10 * a[:, t] * h.abs() + 2 * new.abs())
        h = new
        H[:, t], E[:, t] = h, e
    res = {"output": (torch.where(live, H, 0.0), torch.where(live, E, 0.0)), "state": (h, e)}
    if gy is None:
        return res
    gy = torch.where(live, gy, 0.0)
    g = torch.zeros(B, D, dtype=torch.float64) if gh is None else gh.clone()
    f = torch.zeros_like(g)
    u, F = torch.zeros_like(H), torch.zeros_like(H)
    for t in range(T - 1, -1, -1):
        u[:, t] = gy[:, t] + g
        F[:, t] = f + 2 * U * u[:, t].abs()
        # magnitudes: a sum that cancels was still rounded at the size of its parts
        size = gy[:, t].abs() + g.abs()
        g = a[:, t] * u[:, t]
        f = a[:, t] * (F[:, t] + 14 * U * size)
    d = before - x
    gz = u * d * a * c
    err = a * c * (F * d.abs() + u.abs() * (Eb + U * (before.abs() + x.abs())) + 48 * U * u.abs() * d.abs())
    res["gradX"] = (c * u, c * F + 26 * U * (c * u).abs())
    res["gradGate"] = (gz, err)
    res["gradState"] = (g, f)
    adds = 40 + B * (T // 16 + 1) / 16
    res["gradBias"] = (gz.sum((0, 1)) * factor, abs(factor) * (err.sum((0, 1)) + adds * U * gz.abs().sum((0, 1))))
    return res


def _check(got, want, what):
    value, bound = want
    x = got.detach().cpu().double()
    tol = bound + U * value.abs() + 1e-37
    if got.dtype != torch.float32:
        tol = bound + torch.finfo(got.dtype).eps / 2 * (value.abs() + bound) + (2.0 ** -25 if got.dtype == torch.float16 else 1e-37)
    off = (x - value).abs()
    assert bool((off <= tol).all()), "%s: %g times the bound" % (what, float((off / tol).max()))


def _data(B, T, D, dtype, seed, order="btd"):
    gen = torch.Generator("cuda").manual_seed(seed)
    if order == "bdt":    # steps side by side, as in the planes of a convolution
        make = lambda s=1.0: (torch.randn(B, D, T, generator=gen, device="cuda") * s).to(dtype).transpose(1, 2)   # noqa: E731
    elif order == "tbd":
        make = lambda s=1.0: (torch.randn(T, B, D, generator=gen, device="cuda") * s).to(dtype).transpose(0, 1)   # noqa: E731
    else:
        make = lambda s=1.0: (torch.randn(B, T, D, generator=gen, device="cuda") * s).to(dtype)   # noqa: E731
    from fbcunn_amd import nn
    net = nn.GatedLinearRecurrence(D)
    net.bias.copy_(torch.rand(D, generator=gen, device="cuda") * 6 - 1)
    h0, gh = (torch.randn(B, D, generator=gen, device="cuda") for _ in range(2))
    return net, make(), make(), make(), h0, gh


def _check_all(net, x, gate, gy, h0, gh, lengths=None, factor=1.0):
    want = _plain(x, gate, net.bias, h0, lengths, gy, gh, factor)
    y = net.updateOutput([x, gate], state=h0, lengths=lengths)
    net.backward([x, gate], gy, factor, gradState=gh)
    for name, got in (("output", y), ("state", net.state), ("gradX", net.gradInput[0]), ("gradGate", net.gradInput[1]),
                      ("gradState", net.gradState), ("gradBias", net.gradBias)):
        _check(got, want[name], name)


SHAPES = [(1, 1, 1), (3, 1, 130), (2, 2, 3), (5, 15, 64), (2, 16, 63), (1, 17, 2), (3, 100, 129), (2, 127, 65), (1, 128, 257),
          (4, 129, 515), (2, 255, 1), (1, 256, 128), (3, 300, 33), (1, 1000, 130), (2, 2500, 50), (1, 5000, 7)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%dx%d" % s)
def test_values_and_gradients(shape, dtype):
    _check_all(*_data(*shape, TYPES[dtype], sum(shape)), factor=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(260, 300, 130), (1030, 130, 5)], ids=lambda s: "%dx%dx%d" % s)
def test_one_workgroup_walks_over_the_tiles(shape, dtype):
    data = _data(*shape, TYPES[dtype], 3)
    _check_all(*data)
    assert "chain" not in _lib.lib().fbfc_last_launch().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["bdt", "tbd"])
@pytest.mark.parametrize("shape", [(3, 1, 20), (3, 40, 20), (2, 300, 70)], ids=lambda s: "%dx%dx%d" % s)
def test_other_orders(shape, order):
    _check_all(*_data(*shape, torch.float32, 5, order))


@pytest.mark.gpu
def test_broadcast_gate_and_no_state():
    net, x, gate, gy, _, _ = _data(3, 200, 70, torch.bfloat16, 6)
    want = _plain(x, gate[:1, :1].expand_as(x), net.bias, None, None, gy, None)
    wide = gate[:1, :1].expand_as(x)
    _check(net.updateOutput([x, wide]), want["output"], "output")
    net.backward([x, wide], gy)
    _check(net.gradInput[1], want["gradGate"], "gradGate")
    _check(net.gradState, want["gradState"], "gradState")
    net.bias.zero_()
    want = _plain(x, gate, net.bias)
    _check(net.updateOutput([x, gate]), want["output"], "output")


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 20, 300, 1300])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_padded_batch(T, dtype):
    """Lengths of zero, one, all, and out of range; what lies behind them is no number and is not read."""
    net, x, gate, gy, h0, gh = _data(6, T, 131, TYPES[dtype], 7)
    lengths = torch.tensor([0, 1, T, T - T // 3, T + 5, -2], dtype=torch.int32, device="cuda")
    for b, n in enumerate(lengths.clamp(0, T).tolist()):
        for t, v in ((x, float("nan")), (gate, float("inf")), (gy, float("nan"))):
            t[b, n:] = v
    clean = [torch.nan_to_num(t.float(), 0.0, 0.0, 0.0) for t in (x, gate, gy)]
    want = _plain(clean[0], clean[1], net.bias, h0, lengths, clean[2], gh)
    y = net.updateOutput([x, gate], state=h0, lengths=lengths)
    net.output.fill_(float("nan"))
    y = net.updateOutput([x, gate], state=h0, lengths=lengths)
    net.backward([x, gate], gy, gradState=gh)
    for name, got in (("output", y), ("state", net.state), ("gradX", net.gradInput[0]), ("gradGate", net.gradInput[1]),
                      ("gradState", net.gradState), ("gradBias", net.gradBias)):
        _check(got, want[name], name)
    assert torch.equal(net.state[0], h0[0]) and torch.equal(net.gradState[5], gh[5])


@pytest.mark.gpu
def test_tokens_one_after_the_other():
    net, x, gate, _, h0, _ = _data(5, 40, 300, torch.bfloat16, 8)
    want = _plain(x, gate, net.bias, h0)
    state = h0.clone()
    for t in range(40):
        y = net.step([x[:, t], gate[:, t]], state)
        _check(y, (want["output"][0][:, t], want["output"][1][:, t]), t)
    _check(state, want["state"], "state")
    planes = x[:, :1].transpose(1, 2).contiguous().transpose(1, 2)
    strided = torch.randn(5, 600, device="cuda").bfloat16()[:, ::2]     # channels two apart
    a = net.step([strided, strided], h0.clone())
    b = net.step([strided.contiguous(), strided.contiguous()], h0.clone())
    assert torch.equal(a, b)
    assert torch.equal(net.updateOutput([planes, gate[:, :1]], state=h0), net.updateOutput([x[:, :1], gate[:, :1]], state=h0))


@pytest.mark.gpu
def test_parts_continue_a_sequence():
    """A sequence in two calls, the state handed on in its own place: bit for bit where the cut lies between tiles."""
    net, x, gate, _, h0, _ = _data(2, 1024, 100, torch.float32, 9)
    whole = net.updateOutput([x, gate], state=h0).clone()
    last = net.state.clone()
    first = net.updateOutput([x[:, :512], gate[:, :512]], state=h0).clone()
    second = net.updateOutput([x[:, 512:], gate[:, 512:]], state=net.state)
    want = _plain(x, gate, net.bias, h0)
    _check(torch.cat((first, second), 1), want["output"], "output")
    _check(net.state, want["state"], "state")
    assert torch.equal(first, whole[:, :512]) and last.shape == net.state.shape


@pytest.mark.gpu
def test_no_steps_and_no_sequences():
    net, x, gate, gy, h0, gh = _data(3, 4, 10, torch.float32, 10)
    empty = x[:, :0]
    assert net.updateOutput([empty, empty], state=h0).shape == (3, 0, 10) and torch.equal(net.state, h0)
    net.backward([empty, empty], empty, gradState=gh)
    assert torch.equal(net.gradState, gh) and bool((net.gradBias == 0).all())
    net.updateOutput([empty, empty])
    assert bool((net.state == 0).all())
    net.gradBias.fill_(1.0)
    none = x[:0]
    assert net.updateOutput([none, none]).shape == (0, 4, 10)
    net.backward([none, none], none)
    assert bool((net.gradBias == 0).all())


@pytest.mark.gpu
def test_results_repeat_and_halves_match_the_whole():
    """The state goes from tile to tile through memory in an order that changes from run to run; no result does."""
    net, x, gate, gy, h0, gh = _data(2, 20000, 300, torch.bfloat16, 11)
    results = lambda: [net.output, net.state, *net.gradInput, net.gradState, net.gradBias]   # noqa: E731
    first = None
    for rep in range(4):
        net.updateOutput([x, gate], state=h0)
        if rep == 3:
            net.updateGradInput([x, gate], gy, gh)
            net.gradBias.fill_(float("nan"))
            net.accGradParameters([x, gate], gy, 1.0, gh)
        else:
            net.backward([x, gate], gy, gradState=gh)
        now = [t.clone() for t in results()]
        if first is None:
            first = now
            for t in results():
                t.fill_(float("nan"))
        for a, b in zip(first, now):
            assert torch.equal(a, b), rep


@pytest.mark.gpu
def test_gates_open_and_closed():
    net, x, gate, gy, h0, gh = _data(2, 300, 40, torch.float32, 12)
    gate[0, 5], gate[0, 6], gate[1, 7], gate[1, 8] = float("inf"), -float("inf"), 300.0, -300.0
    y = net.updateOutput([x, gate], state=h0)
    net.backward([x, gate], gy, gradState=gh)
    assert torch.equal(y[0, 5], y[0, 4]) and torch.equal(y[1, 7], y[1, 6])       # kept
    for b, t in ((0, 6), (1, 8)):                                                # replaced: h + (x - h), two roundings
        assert bool(((y[b, t] - x[b, t]).abs() <= 2 * U * (x[b, t].abs() + y[b, t - 1].abs())).all())
    for t in (y, net.state, *net.gradInput, net.gradState, net.gradBias):
        assert bool(t.isfinite().all())
    x[0, 100, 3] = float("nan")                                                  # reaches what follows in its channel alone
    y2 = net.updateOutput([x, gate], state=h0)
    bad = torch.zeros(2, 300, 40, dtype=torch.bool, device="cuda")
    bad[0, 100:, 3] = True
    assert torch.equal(y2.isnan(), bad)


@pytest.mark.gpu
def test_gradient_against_differences():
    """Directional derivative by central differences in 32 bits; the bound is the rounding of the outputs over the step
    and how far the same difference in 64 bits is from the gradient in 64 bits."""
    h = 2.0 ** -5
    net, x, gate, gy, h0, gh = _data(2, 150, 6, torch.float32, 13)
    _, dx, dz, _, dh, _ = _data(2, 150, 6, torch.float32, 14)
    net.updateOutput([x, gate], state=h0)
    net.backward([x, gate], gy, gradState=gh)
    dot = lambda a, b: float((a.detach().cpu().double() * b.detach().cpu().double()).sum())   # noqa: E731
    mine = dot(net.gradInput[0], dx) + dot(net.gradInput[1], dz) + dot(net.gradState, dh)
    want = _plain(x, gate, net.bias, h0, None, gy, gh)
    exact = dot(want["gradX"][0], dx) + dot(want["gradGate"][0], dz) + dot(want["gradState"][0], dh)
    tol = dot(want["gradX"][1], dx.abs()) + dot(want["gradGate"][1], dz.abs()) + dot(want["gradState"][1], dh.abs())
    sums, plain = [], []
    for sign in (1, -1):
        at = [x + sign * h * dx, gate + sign * h * dz]
        y = net.updateOutput(at, state=h0 + sign * h * dh)
        ref = _plain(*at, net.bias, h0 + sign * h * dh)
        sums.append(dot(y, gy) + dot(net.state, gh))
        plain.append(dot(ref["output"][0], gy) + dot(ref["state"][0], gh))
        tol += (dot(ref["output"][1] + U * ref["output"][0].abs(), gy.abs()) + dot(ref["state"][1], gh.abs())) / (2 * h)
    tol += 1.01 * abs((plain[0] - plain[1]) / (2 * h) - exact) + 1e-6 * abs(exact)
    assert abs((sums[0] - sums[1]) / (2 * h) - mine) <= tol
    assert tol < 0.1 * abs(exact)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [100, 1500])
def test_replays_from_a_graph(T):
    net, x, gate, gy, h0, gh = _data(2, T, 200, torch.bfloat16, 15)
    other, *_ = _data(2, T, 200, torch.bfloat16, 15)

    def step(m):
        m.updateOutput([x, gate], state=h0)
        m.backward([x, gate], gy, gradState=gh)

    results = lambda m: [m.output, m.state, *m.gradInput, m.gradState, m.gradBias]   # noqa: E731
    step(net)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(net)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(net)
    for rep in range(3):
        x.mul_(-0.5)
        for t in results(net):
            t.fill_(float("nan"))
        (x.float() * 2).sum().item()
        graph.replay()
        torch.cuda.synchronize()
        step(other)
        for a, b in zip(results(net), results(other)):
            assert torch.equal(a, b), rep


@pytest.mark.gpu
def test_two_streams_at_once():
    """Two long recurrences, each with its workspace, on two streams: neither waits for the other's tiles."""
    jobs = [_data(2, 30000, 200, torch.bfloat16, 16 + i) for i in range(2)]
    want = []
    for net, x, gate, gy, h0, gh in jobs:
        net.updateOutput([x, gate], state=h0)
        net.backward([x, gate], gy, gradState=gh)
        want.append([t.clone() for t in (net.output, *net.gradInput, net.gradBias)])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for rep in range(3):
        for s, (net, x, gate, gy, h0, gh) in zip(streams, jobs):
            with torch.cuda.stream(s):
                net.updateOutput([x, gate], state=h0)
                net.backward([x, gate], gy, gradState=gh)
    torch.cuda.synchronize()
    for (net, *_), w in zip(jobs, want):
        for a, b in zip((net.output, *net.gradInput, net.gradBias), w):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("T,D", [(70016, 32768), (140032, 16384)])    # one workgroup a column; tiles handed on
def test_offsets_beyond_32_bits(T, D):
    """2.3 thousand million elements: the last tiles from the checkpoint before them, as a sequence of their own."""
    from fbcunn_amd import nn
    gen = torch.Generator("cuda").manual_seed(1)
    x, gate = (torch.empty(1, T, D, dtype=torch.bfloat16, device="cuda").normal_(generator=gen) for _ in range(2))
    net = nn.GatedLinearRecurrence(D)
    net.bias.fill_(2.0)
    y = net.updateOutput([x, gate])
    kept = net._forward[3].view(torch.float32)[:T // 128 * D].view(-1, D)
    part = nn.GatedLinearRecurrence(D)
    part.bias.fill_(2.0)
    for cut in (128 * 300, T - 256):
        z = part.updateOutput([x[:, cut:cut + 256], gate[:, cut:cut + 256]], state=kept[cut // 128].view(1, D).contiguous())
        assert torch.equal(z, y[:, cut:cut + 256])
    net.backward([x, gate], y)
    part.backward([x[:, T - 256:], gate[:, T - 256:]], y[:, T - 256:])
    assert torch.equal(net.gradInput[1][:, T - 256:], part.gradInput[1])


@pytest.mark.gpu
def test_module_refusals():
    from fbcunn_amd import nn
    net = nn.GatedLinearRecurrence(8)
    x = torch.randn(2, 5, 8, device="cuda")
    ok = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    for call, error in ((lambda: net.updateOutput([x]), ValueError), (lambda: net.updateOutput([x, x[:1]]), ValueError),
                        (lambda: net.updateOutput([x, x.half()]), TypeError), (lambda: net.updateOutput([x.cpu(), x]), TypeError),
                        (lambda: net.updateOutput([x[..., :4]] * 2), ValueError), (lambda: net.updateOutput([x[0]] * 2), ValueError),
                        (lambda: net.updateOutput([x, x], state=torch.zeros(2, 7, device="cuda")), ValueError),
                        (lambda: net.updateOutput([x, x], state=torch.zeros(2, 8, device="cuda").half()), TypeError),
                        (lambda: net.updateOutput([x, x], lengths=ok.long()), TypeError),
                        (lambda: net.updateOutput([x, x], lengths=ok[:1]), ValueError),
                        (lambda: net.updateOutput([x, x], lengths=ok.cpu()), TypeError),
                        (lambda: net.backward([x, x], x), ValueError),
                        (lambda: net.step([x, x], torch.zeros(2, 8, device="cuda")), ValueError),
                        (lambda: net.step([x[:, 0], x[:, 0]], None), TypeError)):
        with pytest.raises(error):
            call()
    net.updateOutput([x, x], lengths=ok)
    with pytest.raises(ValueError):
        net.backward([x[:1], x[:1]], x[:1])
    net.evaluate()
    net.updateOutput([x, x])
    with pytest.raises(ValueError):
        net.backward([x, x], x)


def test_misaligned_states_and_oversized_shapes_are_refused():
    for kw in (dict(bias=0x1002), dict(state_in=0x1001), dict(lengths=0x1002), dict(state_out=0x1002), dict(checkpoints=0x1003)):
        rc, message = _forward(**kw)
        assert rc == _lib.ERR_INVALID_ARGUMENT and "4 bytes" in message
    for kw in (dict(bias=0x1002), dict(lengths=0x1001), dict(checkpoints=0x1002), dict(gstate=0x1002), dict(gb=0x1002), dict(gstate_in=0x1001)):
        rc, message = _backward(**kw)
        assert rc == _lib.ERR_INVALID_ARGUMENT and "4 bytes" in message
    # one launch has fewer than 2^32 threads
    for kw in (dict(channels=(1 << 25) + 1), dict(batch=1 << 16, channels=1 << 15), dict(batch=1 << 23, channels=1),
               dict(batch=1, channels=64, steps=1 << 31)):
        assert _forward(**kw)[0] == _lib.ERR_UNSUPPORTED_SIZE, kw


@pytest.mark.gpu
def test_own_output_as_input_keeps_its_values():
    """A module whose last output is its next input: the output goes elsewhere, and backward sees the input."""
    net, x, gate, gy, _, _ = _data(2, 200, 12, torch.float32, 17)
    y = net.updateOutput([x, gate])
    kept = y.clone()
    z = net.updateOutput([y, gate])
    assert z is not y and torch.equal(y, kept)
    net.backward([y, gate], gy)
    want = _plain(kept, gate, net.bias, None, None, gy, None)
    _check(z, want["output"], "output")
    _check(net.gradInput[1], want["gradGate"], "gradGate")


def test_sizes_that_no_launch_takes_are_refused_with_no_sequences_too():
    # the sum of the bias's gradient has 64 threads for each channel, whatever the batch
    assert _backward(batch=0, channels=1 << 27, gb=P)[0] == _lib.ERR_UNSUPPORTED_SIZE
    # 256 columns of one channel a lane, and 128 of two: there each tile is a workgroup
    assert _forward(batch=1, channels=64 * 256, steps=1 << 31, type=_lib.BF16)[0] == _lib.ERR_UNSUPPORTED_SIZE


@pytest.mark.gpu
def test_parameters_on_another_device_are_refused():
    from fbcunn_amd import nn
    net = nn.GatedLinearRecurrence(8, device="cpu")
    x = torch.randn(2, 5, 8, device="cuda")
    with pytest.raises(ValueError, match="another device"):
        net.updateOutput([x, x])
    with pytest.raises(ValueError, match="another device"):
        net.step([x[:, 0], x[:, 0]], torch.zeros(2, 8, device="cuda"))


@pytest.mark.gpu
def test_views_of_the_own_output_as_input_keep_their_values():
    from fbcunn_amd import nn
    net, x, gate, gy, _, _ = _data(6, 6, 12, torch.float32, 18)
    y = net.updateOutput([x, gate])
    turned, kept = y.transpose(0, 1), y.clone()      # the same shape, other strides
    z = net.updateOutput([turned, gate])
    assert z is not y and torch.equal(y, kept)
    net.backward([turned, gate], gy)
    want = _plain(kept.transpose(0, 1), gate, net.bias, None, None, gy, None)
    _check(z, want["output"], "output")
    _check(net.gradInput[1], want["gradGate"], "gradGate")
    # a token of two sequences, swapped
    net = nn.GatedLinearRecurrence(12)
    a, state = net.step([x[:2, 0], gate[:2, 0]], torch.zeros(2, 12, device="cuda")), torch.zeros(2, 12, device="cuda")
    kept = a.clone()
    b = net.step([a[:, :], a], state)
    want = _plain(kept[:, None], kept[:, None], net.bias, None, None, kept[:, None], None)
    assert b is not a and torch.equal(a, kept)
    _check(b[:, None], want["output"], "output")


@pytest.mark.gpu
def test_a_graph_keeps_its_results_when_the_module_goes_on_with_other_shapes():
    net, x, gate, gy, h0, gh = _data(2, 150, 40, torch.float32, 19)
    other, *_ = _data(2, 150, 40, torch.float32, 19)

    def step(m, n=150):
        m.updateOutput([x[:, :n], gate[:, :n]], state=h0)
        m.backward([x[:, :n], gate[:, :n]], gy[:, :n], gradState=gh)

    step(net)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(net)
    y = net.output
    for n in (70, 150, 3):
        step(net, n)
    # memory that the module has given back would be found here
    fill = [torch.full((k,), 7.0, device="cuda") for k in (80, 2 * 150 * 40) for _ in range(20)]
    for rep in range(3):
        x.mul_(-0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(bool((t == 7.0).all()) for t in fill)
        step(other)
        assert torch.equal(y, other.output) and torch.equal(net.gradBias, other.gradBias)


@pytest.mark.gpu
def test_a_captured_step_is_a_new_token_at_each_replay():
    net, x, gate, _, h0, _ = _data(5, 7, 70, torch.bfloat16, 20)
    other, *_ = _data(5, 7, 70, torch.bfloat16, 20)
    state, want = h0.clone(), h0.clone()
    at, to = x[:, 0].clone(), gate[:, 0].clone()
    net.step([at, to], state.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = net.step([at, to], state)
    for t in range(7):
        at.copy_(x[:, t])
        to.copy_(gate[:, t])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, other.step([x[:, t], gate[:, t]], want)) and torch.equal(state, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("planes", ["inputs", "gradient", "all", "x"])
@pytest.mark.parametrize("shape", [(1, 16, 64), (2, 47, 70), (3, 300, 130), (2, 1500, 33), (300, 40, 1)], ids=lambda s: "%dx%dx%d" % s)
def test_planes_of_a_convolution_beside_rows_of_channels(shape, planes, dtype):
    net, x, gate, gy, h0, gh = _data(*shape, TYPES[dtype], 21)
    turn = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)   # noqa: E731
    if planes != "gradient":
        x = turn(x)
    if planes in ("inputs", "all"):
        gate = turn(gate)
    if planes in ("gradient", "all"):
        gy = turn(gy)
    _check_all(net, x, gate, gy, h0, gh)
    lengths = torch.arange(shape[0], dtype=torch.int32, device="cuda") * 17 % (shape[1] + 1)
    _check_all(net, x, gate, gy, h0, gh, lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [300, 2500])
def test_one_module_in_two_graphs_and_on_two_streams_at_once(T):
    """The tiles of a call wait for each other through the workspace: calls that may run at the same time have one each."""
    net, x, gate, gy, h0, gh = _data(2, T, 70, torch.float32, 22)

    def step():
        net.updateOutput([x, gate], state=h0)
        net.backward([x, gate], gy, gradState=gh)

    step()
    results = [net.output, net.state, *net.gradInput, net.gradState, net.gradBias]
    want = [t.clone() for t in results]
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g in graphs:
        with torch.cuda.graph(g):
            step()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        with torch.cuda.stream(s):
            step()
    torch.cuda.synchronize()
    used = [w.data_ptr() for w in net._workspace._captured] + [w.data_ptr() for w in net._workspace._of.values()]
    assert len(used) == len(set(used)) == 2 * 2 + 3
    for rep in range(3):
        for t in results:
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):   # the same inputs and results, so they agree whatever runs first
            with torch.cuda.stream(s):
                g.replay()
        step()
        for s in streams:
            with torch.cuda.stream(s):
                step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(results, want)), rep


def _closed(dtype):
    """Gates that replace the state, or keep it: around where e^z leaves the normal numbers, and far beyond."""
    return [-80.0, -86.0, -87.0, -88.0, -104.0, -300.0, torch.finfo(dtype).min, -float("inf"), 88.0, 300.0, float("inf")]


def _close(gate, T):
    """Channel (i, j) of `gate` has value i of _closed() at place j: the ends of a run of 16 steps, of a tile of 128, of the
    sequence, their neighbours, and a whole run.  {place: steps}"""
    places = [[t] for t in (0, 1, 15, 16, 40, 127, 128, T - 1) if t < T] + [list(range(32, 48))] * (T >= 48)
    values = _closed(gate.dtype)
    for j, steps in enumerate(places):
        for i, v in enumerate(values):
            gate[:, steps, j * len(values) + i] = v
    return places


@pytest.mark.gpu
@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape,order", [((2, 1, 25), "btd"), ((3, 16, 45), "btd"), ((2, 300, 101), "btd"), ((3, 700, 101), "bdt"),
                                         ((2, 300, 101), "tbd"), ((130, 300, 101), "btd")], ids=str)
def test_gradients_at_closed_gates(shape, order, dtype, padded):
    """The bounds of _plain() hold for gates below 10.  At the others here the smaller of a and 1 - a is below 2e-35.  Its relative
    error is below 2^-15: |z| + 2 units of 2^-24 for up to 104, and zero in its place below 2^-126.  So it is off by less than 2^-126,
    and a result, which is a sum of at most B T products of it with one u and one d, by less than 2^-126 B T |u| |d|, where
    |u| <= |gh| + T max |gy|, and |d| <= 2 max(|x|, |h0|) because a state lies between those."""
    net, x, gate, gy, h0, gh = _data(*shape, TYPES[dtype], 23, order)
    net.bias.zero_()
    _close(gate, shape[1])
    lengths = None
    if padded:   # the full length, one step less, which ends before the gate of the last one, and so on
        lengths = (shape[1] - torch.arange(shape[0], device="cuda") % 3 * (shape[1] // 3)).to(torch.int32)
        lengths[1] = shape[1] - 1
    want = _plain(x, gate, net.bias, h0, lengths, gy, gh)
    top = lambda *t: max(1.0, *(float(v.abs().max()) for v in t))   # noqa: E731
    under = 2.0 ** -126 * shape[0] * shape[1] * (shape[1] + 1) * top(gy, gh) * 2 * top(x, h0)
    assert under < 1e-28   # nothing beside the other roundings
    y = net.updateOutput([x, gate], state=h0, lengths=lengths)
    net.backward([x, gate], gy, gradState=gh)
    for name, got in (("output", y), ("state", net.state), ("gradX", net.gradInput[0]), ("gradGate", net.gradInput[1]),
                      ("gradState", net.gradState), ("gradBias", net.gradBias)):
        _check(got, (want[name][0], want[name][1] + under), name)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 300, 101), (130, 300, 101)], ids=str)
def test_no_gradient_passes_a_closed_gate(shape):
    net, x, gate, gy, h0, gh = _data(*shape, torch.float32, 24)
    net.bias.zero_()
    values, places = _closed(torch.float32), _close(gate, shape[1])
    net.updateOutput([x, gate], state=h0)
    first = [t.clone() for t in net.backward([x, gate], gy, gradState=gh)] + [net.gradState.clone()]
    after = torch.zeros(shape, dtype=torch.bool, device="cuda")
    for j, steps in enumerate(places):
        for i, v in enumerate(values):
            if v <= -104:
                after[:, steps[-1]:, j * len(values) + i] = True
    other = torch.where(after, gy * 2 + 1, gy)
    again = net.backward([x, gate], other, gradState=torch.where(after[:, -1], gh * 2 + 1, gh)) + [net.gradState]
    for a, b in zip(first[:2], again[:2]):   # of the steps before the gate
        assert torch.equal(torch.where(after, 0, a), torch.where(after, 0, b))
    closed = after.any(1)
    assert torch.equal(first[2][closed], again[2][closed])
    assert not torch.equal(first[0], again[0])


def test_a_result_that_a_graph_writes_to_is_kept_when_another_takes_its_place():
    import weakref
    from fbcunn_amd.sequence import _Call
    call = _Call(torch.zeros(4, 5), 1)
    alive = lambda refs: [r() is not None for r in refs]   # noqa: E731
    first = call.result(0)
    call.captured = call.capturing = True
    assert call.result(0) is first                       # made before the capture, written in it
    second = call.result(0, [first.data_ptr()])          # an input of the captured call itself
    call.capturing = False
    third = call.result(0, [second.data_ptr()])          # an input of a later call
    fourth = call.result(0, [third.data_ptr() + 4])      # no graph writes to the third
    refs = [weakref.ref(t) for t in (first, second, third, fourth)]
    del first, second, third, fourth
    assert alive(refs) == [True, True, False, True]


@pytest.mark.gpu
@pytest.mark.parametrize("twice", [True, False])
def test_a_graph_keeps_results_that_were_its_modules_inputs(twice):
    """A module applied twice in a captured step, or eagerly to what a captured step gave; all references dropped, memory
    that was given back would be found by the fill."""
    net, x, gate, *_ = _data(2, 150, 40, torch.float32, 25)
    other, *_ = _data(2, 150, 40, torch.float32, 25)
    apply = lambda m: m.updateOutput([m.updateOutput([x, gate]) if twice else x, gate])   # noqa: E731
    apply(net)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = apply(net)
    if not twice:
        net.updateOutput([net.updateOutput([y, gate]), gate])
    seen = y.data_ptr()
    del y
    fill = [torch.full((2 * 150 * 40,), 7.0, device="cuda") for _ in range(40)]
    assert seen not in [t.data_ptr() for t in fill]
    for rep in range(3):
        x.mul_(-0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(bool((t == 7.0).all()) for t in fill), rep
        apply(other)


def _same(net, other, what):
    results = lambda m: [m.output, m.state, *m.gradInput, m.gradState, m.gradBias]   # noqa: E731
    for i, (a, b) in enumerate(zip(results(net), results(other))):
        assert torch.equal(a, b), (what, i)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [40, 700])
def test_own_gradients_and_states_as_inputs_keep_their_values(T):
    """What the module's last call gave is an input of the next, whose halves both have to find it as it was."""
    net, x, gate, gy, h0, gh = _data(2, T, 40, torch.float32, 26)
    other, *_ = _data(2, T, 40, torch.float32, 26)

    def halves(m, inputs, grad):
        m.updateOutput(inputs, state=h0)
        m.updateGradInput(inputs, grad, gh)
        m.accGradParameters(inputs, grad, 1.0, gh)

    halves(net, [x, gate], gy)
    for i in range(2):
        mine = net.gradInput[i]
        kept = mine.clone()
        halves(net, [x, gate], mine)         # a gradient of the output
        halves(other, [x, gate], kept)
        assert torch.equal(mine, kept)
        _same(net, other, ("gradOutput", i))
        mine = net.gradInput[i]
        kept = mine.clone()
        halves(net, [mine, gate], gy)        # an input
        halves(other, [kept, gate], gy)
        assert torch.equal(mine, kept)
        _same(net, other, ("input", i))
    mine = net.gradState
    kept = mine.clone()
    net.updateGradInput([x, gate], gy, mine), net.accGradParameters([x, gate], gy, 1.0, mine)
    other.updateGradInput([x, gate], gy, kept), other.accGradParameters([x, gate], gy, 1.0, kept)
    assert torch.equal(mine, kept)
    _same(net, other, "gradState")
    last = lambda m: m.updateOutput([x[:, :1], gate[:, :1]], state=h0)   # noqa: E731
    last(net), last(other)
    for name in ("state", "state", "gradState"):           # a state as a sequence of one step
        mine = getattr(net, name)
        kept = mine.clone()
        halves(net, [mine[:, None], gate[:, :1]], gy[:, :1])
        halves(other, [kept[:, None], gate[:, :1]], gy[:, :1])
        assert torch.equal(mine, kept)
        _same(net, other, name)


def test_parameters_are_looked_at_in_each_call():
    """An address goes on only of as many 32-bit numbers, side by side, on the inputs' device."""
    from fbcunn_amd.sequence import _parameter
    t = torch.zeros(8)
    assert _parameter(t, "bias", 8, -1) == t.data_ptr() and _parameter(None, "bias", 8, -1) is None
    for bad, index, error, text in ((t[:7], -1, ValueError, "8 contiguous"), (torch.zeros(9), -1, ValueError, "8 contiguous"),
                                    (torch.zeros(16)[::2], -1, ValueError, "8 contiguous"), (t.half(), -1, TypeError, "float32"),
                                    (t.double(), -1, TypeError, "float32"), (t, 0, ValueError, "another device"), ([0.0] * 8, -1, TypeError, "tensor")):
        with pytest.raises(error, match=text):
            _parameter(bad, "bias", 8, index)


@pytest.mark.gpu
def test_parameters_that_do_not_fit_are_refused():
    net, x, gate, gy, h0, _ = _data(2, 5, 8, torch.float32, 27)
    net.updateOutput([x, gate])
    net.backward([x, gate], gy)
    net.step([x[:, 0], gate[:, 0]], h0)
    whole = net.bias, net.gradBias
    for bad, error in ((whole[0].half(), TypeError), (whole[0][:7], ValueError), (whole[0].cpu(), ValueError)):
        net.bias = bad
        for call in (lambda: net.updateOutput([x, gate]), lambda: net.backward([x, gate], gy), lambda: net.step([x[:, 0], gate[:, 0]], h0)):
            with pytest.raises(error, match="bias"):
                call()
        net.bias, net.gradBias = whole[0], bad
        net.updateOutput([x, gate])
        net.updateGradInput([x, gate], gy)
        for call in (lambda: net.backward([x, gate], gy), lambda: net.accGradParameters([x, gate], gy)):
            with pytest.raises(error, match="gradBias"):
                call()
        net.gradBias = whole[1]
    net.bias.data = net.bias.data.half()       # the same tensor, of another type
    with pytest.raises(TypeError, match="bias"):
        net.updateOutput([x, gate])


def _lerp_bound(z, x, h, new):
    """Of one step, with z the gate: the smaller of a and 1 - a comes from e^-|z|, whose argument is rounded twice (2 |z| units),
    with 8 units for exponential, sum, reciprocal and product; the larger is one minus that.  The state moves from the side
    with the larger weight, so the difference's rounding counts with the smaller one."""
    a, c = torch.sigmoid(z), torch.sigmoid(-z)
    return U * (torch.minimum(a, c) * (2 * z.abs() + 12) * (x.abs() + h.abs()) + 2 * new.abs())


def _large_state(B, T, dtype, order, seed):
    """States a million times the inputs, kept as they are up to the middle, where gates from half closed to closed follow, the
    first four closed for good; kept again behind it."""
    net, x, gate, gy, h0, gh = _data(B, T, 60, dtype, seed, order)
    net.bias.zero_()
    at = T // 2
    gate[:, :at], gate[:, at:] = float("inf"), 88.0
    gate[:, at] = -torch.linspace(0, 40, 60, device="cuda").to(dtype)
    gate[:, at, :4] = torch.tensor([-104.0, -300.0, torch.finfo(dtype).min, -float("inf")], device="cuda").to(dtype)
    return net, x, gate, gy, h0 * 1e6, gh, at


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,order", [(1, "btd"), (24, "btd"), (500, "btd"), (500, "bdt")])
def test_a_large_state_leaves_no_rounding_behind_a_closed_gate(T, order, dtype):
    """What is left of the state is its weight's part, and nothing rounded at the state's size; behind a gate that is closed for
    good the state is the input itself."""
    net, x, gate, _, h0, _, at = _large_state(3, T, TYPES[dtype], order, 28)
    z, v, h = gate[:, at].cpu().double().clamp(min=-1000), x[:, at].cpu().double(), h0.cpu().double()
    want = torch.sigmoid(z) * h + torch.sigmoid(-z) * v
    bound = _lerp_bound(z, v, h, want)
    y = net.updateOutput([x, gate], state=h0)
    if dtype != "f16":     # 1e6 is beyond its numbers
        _check(y[:, at], (want, bound), "output")
    _check(net.state, (want, bound), "state")
    assert torch.equal(y[:, at, :4], x[:, at, :4]) and torch.equal(net.state[:, :4], x[:, at, :4].float())
    state = h0.clone()
    token = net.step([x[:, at], gate[:, at]], state)
    _check(state, (want, bound), "state of a token")
    assert torch.equal(state[:, :4], x[:, at, :4].float()) and torch.equal(token[:, :4], x[:, at, :4])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,order", [(24, "btd"), (500, "btd"), (500, "bdt")])
def test_backward_forms_the_state_behind_a_closed_gate_as_forward_does(T, order, dtype):
    """The gate behind the closed one is half open: its gradient is u (state - x) / 4, the state the closed one's input.  u is a sum
    of at most T + 1 numbers, rounded T times, and 12 units are left for the weights, the difference and the products."""
    net, x, gate, gy, h0, gh, at = _large_state(3, T, TYPES[dtype], order, 29)
    gate[:, at + 1] = 0.0
    net.updateOutput([x, gate], state=h0)
    net.backward([x, gate], gy, gradState=gh)
    x, gy, gh = x.cpu().double(), gy.cpu().double(), gh.cpu().double()
    d = x[:, at] - x[:, at + 1]
    u, size = gh + gy[:, at + 1:].sum(1), gh.abs() + gy[:, at + 1:].abs().sum(1)
    _check(net.gradInput[1][:, at + 1, :4], ((u * d / 4)[:, :4], (U * (T + 12) * size * d.abs() / 4)[:, :4]), "gradGate")


def test_buffers_of_an_unused_module_are_cleaned_up_without_a_gpu():
    from fbcunn_amd import nn
    for net in (nn.GatedLinearRecurrence(8, device="cpu"), nn.GatedResidualNorm(8, device="cpu")):
        net.cleanupBuffers()


@pytest.mark.gpu
def test_cleanup_gives_back_what_captured_calls_took():
    """Graphs for one length after the other: what they held goes with cleanupBuffers(), after which the module works on."""
    net, x, gate, gy, h0, gh = _data(2, 3000, 200, torch.float32, 30)
    other, *_ = _data(2, 3000, 200, torch.float32, 30)

    def step(m, n):
        m.updateOutput([x[:, :n], gate[:, :n]], state=h0)
        m.backward([x[:, :n], gate[:, :n]], gy[:, :n], gradState=gh)

    step(other, 3000)
    step(net, 10)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    before = torch.cuda.memory_allocated()
    for n in (500, 1000, 2000, 3000):
        step(net, n)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(net, n)
        graph.replay()
        torch.cuda.synchronize()
        del graph
    held = torch.cuda.memory_allocated()
    last = [net.output, net.state, *net.gradInput, net.gradState]
    net.cleanupBuffers()
    assert all(torch.equal(a, b) for a, b in zip(last, [other.output, other.state, *other.gradInput, other.gradState]))
    assert held - torch.cuda.memory_allocated() > 3 * sum(n * 2 * 200 * 4 for n in (500, 1000, 2000))
    del last
    net.output = net.state = net.gradInput = net.gradState = None
    assert torch.cuda.memory_allocated() <= before
    with pytest.raises(ValueError):
        net.backward([x, gate], gy)       # follows an updateOutput
    step(net, 3000)
    _same(net, other, "after")


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 40, 700])
def test_a_state_that_is_a_row_of_the_own_output_keeps_its_values(T):
    """One sequence in parts, each from the last output of the part before, which is needed again."""
    net, x, gate, gy, h0, _ = _data(1, T, 40, torch.float32, 31)
    other, *_ = _data(1, T, 40, torch.float32, 31)
    first = net.updateOutput([x, gate], state=h0)
    kept = first.clone()
    net.updateOutput([x, gate], state=first[:, -1])
    other.updateOutput([x, gate], state=kept[:, -1])
    assert torch.equal(first, kept)
    net.backward([x, gate], gy, gradState=first[:, 0])
    other.backward([x, gate], gy, gradState=kept[:, 0])
    _same(net, other, "output")
    first = net.gradInput[0]
    kept = first.clone()
    net.backward([x, gate], gy, gradState=first[:, 0])
    other.backward([x, gate], gy, gradState=kept[:, 0])
    assert torch.equal(first, kept)
    _same(net, other, "gradInput")
