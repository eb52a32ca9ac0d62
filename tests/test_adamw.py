"""The AdamW step over many tensors (optim.AdamW, fbfc_adamw_*): against the formulas in 64 bits, and the 8-bit states against
a plain evaluation of their definition, bit for bit."""
import ctypes
import math

import pytest
import torch

from fbcunn_amd import _lib

U = 2.0 ** -24
K1, K2, K3 = 0x9E3779B1, 0xBB67AE85, 0xB504F335
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HYPER = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weightDecay=0.1)


# refusals: no GPU needed ------------------------------------------------------------------------------

def _config(**kw):
    d = dict(param_type=0, grad_type=0, state_bits=32, seed=0, beta1=0.9, beta2=0.99, eps=1e-8)
    d.update(kw)
    return _lib.AdamwConfig(**d)


def _create(config, tensors, m=0x100000, v=0x200000, ms=0x300000, vs=0x400000):
    table = (_lib.AdamwTensor * max(1, len(tensors)))(*tensors)
    h = ctypes.c_void_p(0)
    rc = _lib.lib().fbfc_adamw_create(ctypes.byref(config), table, len(tensors), m, v, ms, vs, ctypes.byref(h))
    assert not h.value
    return rc, _lib.lib().fbfc_last_error().decode()


@pytest.mark.parametrize("config,tensors,text", [
    ({}, [], "at least one"),
    (dict(param_type=3), [(0x1000, 0x2000, 8)], "type"),
    (dict(grad_type=-1), [(0x1000, 0x2000, 8)], "type"),
    (dict(state_bits=16), [(0x1000, 0x2000, 8)], "8 or 32"),
    (dict(beta1=1.0), [(0x1000, 0x2000, 8)], "betas"),
    (dict(beta2=-0.1), [(0x1000, 0x2000, 8)], "betas"),
    (dict(beta1=float("nan")), [(0x1000, 0x2000, 8)], "betas"),
    (dict(eps=0.0), [(0x1000, 0x2000, 8)], "eps"),
    (dict(eps=1e-60), [(0x1000, 0x2000, 8)], "eps"),     # zero in 32 bits
    ({}, [(0x1000, 0x2000, -1)], "negative"),
    ({}, [(0, 0x2000, 8)], "null"),
    ({}, [(0x1000, 0, 8)], "null"),
    ({}, [(0x1002, 0x2000, 8)], "aligned"),
    ({}, [(0x1000, 0x2001, 8)], "aligned"),
    ({}, [(0x1000, 0x2000, 8), (0x101c, 0x3000, 8)], "shares memory"),      # the last float of the first tensor
    ({}, [(0x1000, 0x2000, 8), (0x1000, 0x3000, 8)], "shares memory"),      # the same tensor twice
    ({}, [(0x1000, 0x1000, 8)], "shares memory"),                            # a gradient that is its parameter
    ({}, [(0x100000, 0x2000, 8)], "shares memory"),                          # a parameter in the states
])
def test_refusals(config, tensors, text):
    rc, message = _create(_config(**config), tensors)
    assert rc == _lib.ERR_INVALID_ARGUMENT and text in message, message


def test_refusals_of_states_and_handles():
    good = [(0x1000, 0x2000, 8)]
    for kw, text in ((dict(m=0), "null"), (dict(v=0), "null"), (dict(m=0x100008), "16-byte"), (dict(v=0x200004), "16-byte")):
        rc, message = _create(_config(), good, **kw)
        assert rc == _lib.ERR_INVALID_ARGUMENT and text in message
    rc, message = _create(_config(state_bits=8), good, ms=0)
    assert rc == _lib.ERR_INVALID_ARGUMENT and "scales" in message
    rc, message = _create(_config(state_bits=8), good, vs=0x100000)
    assert rc == _lib.ERR_INVALID_ARGUMENT and "shares memory" in message
    rc, _ = _create(_config(), [(0x1000, 0x2000, 1 << 41)])
    assert rc == _lib.ERR_UNSUPPORTED_SIZE
    L, n = _lib.lib(), ctypes.c_long(0)
    assert L.fbfc_adamw_step(None, 1e-3, 0.0, 1.0, None) == _lib.ERR_INVALID_ARGUMENT
    assert L.fbfc_adamw_set_step(None, 0, None) == _lib.ERR_INVALID_ARGUMENT
    assert L.fbfc_adamw_get_step(None, ctypes.byref(n), None) == _lib.ERR_INVALID_ARGUMENT
    assert L.fbfc_adamw_destroy(None) == _lib.OK


def test_gradients_may_be_shared_and_states_are_counted_in_blocks():
    table = (_lib.AdamwTensor * 3)((0x1000, 0x2000, 1), (0x3000, 0x2000, 256), (0x5000, 0x2000, 257))
    assert _lib.lib().fbfc_adamw_state_elements(table, 3) == 256 + 256 + 512
    assert _lib.lib().fbfc_adamw_state_elements(table, 0) == 0


def test_module_refuses_what_is_not_on_the_gpu():
    from fbcunn_amd import optim
    with pytest.raises(TypeError):
        optim.AdamW([torch.zeros(3)], [torch.zeros(3)])
    with pytest.raises(ValueError):
        optim.AdamW([], [])


# plain forms ---------------------------------------------------------------------------------------------

def _blocks(tensors):
    """The tensors one after the other in 64 bits, each filled up to whole blocks."""
    return torch.cat([torch.nn.functional.pad(t.detach().cpu().double().reshape(-1), (0, -t.numel() % 256)) for t in tensors])


def _random(n, key):
    i, low = torch.arange(n), 0xFFFFFFFF
    x = ((i & low) * K1 + (i >> 32) * K3 + key) & low
    x ^= x >> 16
    x = (x * K2) & low
    x ^= x >> 15
    x = (x * K3) & low
    x ^= x >> 16
    y = (x * K1) & low
    y ^= y >> 16
    y = (y * K2) & low
    return (x >> 12).int(), (y >> 12).int()


def _round8(x, random, positive):
    x = x.view(-1, 256)
    top = x.abs().amax(1)
    scale = torch.where(top < 2.0 ** -100, torch.zeros(()), top * (1 / 448))
    inverse = torch.where(scale > 0, 1 / scale, torch.zeros(()))[:, None]
    bits = (x.abs() * inverse * 2.0 ** -120).view(torch.int32)
    code = ((bits + random.view(-1, 256)) >> 20).clamp(max=0x7E)
    if positive:
        code = torch.where((code == 0) & (x > 0) & (inverse > 0), 1, code)
    else:
        code = code | ((x < 0).int() << 7)
    return code.to(torch.uint8).view(-1), scale


def _value(codes, scale):
    return (codes.cpu().view(torch.float8_e4m3fn).float().view(-1, 256) * scale.cpu()[:, None]).view(-1)


class Plain:
    """The step in 64 bits, from the values that the optimizer held before it."""

    def __init__(self, opt, seed=0):
        self.opt, self.t, self.seed = opt, opt.t, seed

    def states(self):
        o = self.opt
        if o.stateBits == 32:
            return o.m.cpu().clone(), o.v.cpu().clone()
        return _value(o.m, o.mScale), _value(o.v, o.vScale)

    def step(self, run, scale=1.0):
        """Runs one step and checks parameters and states."""
        o, self.t = self.opt, self.t + 1
        (b1, b2) = HYPER["betas"]
        m0, v0 = self.states()
        p0, g = _blocks(o.params), _blocks(o.grads) * scale
        run()
        torch.cuda.synchronize()
        take = m0.double().abs() * b1 + g.abs() * (1 - b1)
        m, v = m0.double() * b1 + g * (1 - b1), v0.double() * b2 + g * g * (1 - b2)
        d = (v / (1 - b2 ** self.t)).sqrt() + HYPER["eps"]
        step = HYPER["lr"] / (1 - b1 ** self.t)
        p = p0 * (1 - HYPER["lr"] * HYPER["weightDecay"]) - step * m / d
        got, kind = _blocks(o.params), o.params[0].dtype
        # 3 roundings of the product with the decay, 16 of the quotient whose numerator is a sum of `take`; half a
        # spacing of the parameters' type
        tol = U * (3 * p0.abs() + 16 * step * take / d) + 1e-40
        if kind != torch.float32:
            tol = tol + torch.finfo(kind).eps / 2 * (p.abs() + tol) + (2.0 ** -25 if kind == torch.float16 else 0)
        assert bool(((got - p).abs() <= tol).all()), float(((got - p).abs() / tol).max())
        if o.stateBits == 32:
            assert bool(((o.m.cpu().double() - m).abs() <= 5 * U * take + 1e-44).all())
            assert bool(((o.v.cpu().double() - v).abs() <= 6 * U * v + 1e-44).all())
            return
        # 8 bits: the same bits as the plain evaluation in 32, and at most one spacing from the value in 64
        r = _random(m.numel(), (self.seed * K1 + self.t * K2) & 0xFFFFFFFF)
        g32 = g.float()
        m32 = m0 * b1 + g32 * (1 - b1)
        v32 = v0 * b2 + g32 * g32 * (1 - b2)
        for x, exact, codes, scales, random, positive in ((m32, m, o.m, o.mScale, r[0], False), (v32, v, o.v, o.vScale, r[1], True)):
            want, scale = _round8(x, random, positive)
            assert torch.equal(scale, scales.cpu())
            assert torch.equal(want, codes.cpu().view(torch.uint8))
            unit = scales.cpu().double().repeat_interleave(256)
            y = exact.abs() / unit.clamp(min=1e-40)
            gap = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
            off = (_value(codes, scales).double() - exact).abs()
            assert bool((off <= unit * gap * (1 + 1e-4) + 2.0 ** -99).all())


def _tensors(sizes, param, grad, packed, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    out = []
    for kind, size in ((param, 0.05), (grad, 0.01)):
        at = 3 if packed else 0
        total = sum(n if packed else -(-n // 64) * 64 for n in sizes) + 64
        flat = (torch.randn(total, generator=g, device="cuda") * size).to(TYPES[kind])
        views = []
        for n in sizes:
            views.append(flat[at:at + n])
            at += n if packed else -(-n // 64) * 64
        out.append((flat, views))
    return out


SIZES = [[1], [255, 256, 257], [4095, 4096, 4097, 3], [0, 5, 0, 1023, 0], [8192 + 7], [(i * 37) % 501 for i in range(300)], [70001, 2, 33333]]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("param,grad,packed", [("f32", "f32", False), ("f32", "f32", True), ("f32", "bf16", True), ("bf16", "bf16", True),
                                               ("f16", "f16", False), ("bf16", "f32", False), ("f32", "f16", True), ("f16", "bf16", True), ("bf16", "f16", True)])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "%dx%d" % (len(s), max(s)))
def test_steps_follow_the_formula(sizes, param, grad, packed, bits):
    from fbcunn_amd import optim
    (pf, params), (gf, grads) = _tensors(sizes, param, grad, packed, 7)
    before, where = pf.clone(), torch.zeros_like(pf, dtype=torch.bool)
    base = pf.data_ptr()
    for t in params:
        if t.numel():
            o = (t.data_ptr() - base) // t.element_size()
            where[o:o + t.numel()] = True
    opt = optim.AdamW(params, grads, stateBits=bits, seed=5, **HYPER)
    plain = Plain(opt, 5)
    for k in range(3):
        plain.step(lambda: opt.step(0.5 if k == 1 else 1.0), 0.5 if k == 1 else 1.0)
        gf.copy_((gf.float() * -0.7 + 0.001).to(gf.dtype))
    assert opt.t == 3
    assert torch.equal(pf[~where], before[~where])   # nothing beside the tensors is written


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_step_on_another_stream_replays_from_a_graph(bits):
    """Every replay is the next step: three replays equal three eager steps bit for bit."""
    from fbcunn_amd import optim
    sizes = [1000, 3, 5000]
    kw = dict(stateBits=bits, seed=9, **HYPER)
    (pf, params), (gf, grads) = _tensors(sizes, "f32", "f32", False, 3)
    (qf, others), (hf, hs) = _tensors(sizes, "f32", "f32", False, 3)
    a, b = optim.AdamW(params, grads, **kw), optim.AdamW(others, hs, **kw)
    a.step(), b.step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step(), b.step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for rep in range(3):
        for f in (gf, hf):
            f.mul_(-0.9)
        (gf * 2).sum().item()
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        assert torch.equal(pf, qf), rep
        for x, y in ((a.m, b.m), (a.v, b.v)):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert a.t == b.t == 5


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_stored_states_continue_the_run(bits):
    from fbcunn_amd import optim
    kw = dict(stateBits=bits, seed=2, **HYPER)
    (pf, params), (_, grads) = _tensors([300, 4097], "f32", "bf16", True, 4)
    a = optim.AdamW(params, grads, **kw)
    a.step(), a.step()
    qf = pf.clone()
    others = [qf[t.storage_offset():t.storage_offset() + t.numel()] for t in params]
    b = optim.AdamW(others, grads, **kw)
    b.loadState(a.m, a.v, a.mScale, a.vScale, a.t)
    a.step(), b.step()
    assert torch.equal(pf, qf) and torch.equal(a.v.view(torch.uint8), b.v.view(torch.uint8)) and b.t == 3
    with pytest.raises(ValueError):
        b.loadState(a.m[:256], a.v, a.mScale, a.vScale, 0)
    with pytest.raises(ValueError):
        b.loadState(a.m, a.v, None if bits == 8 else a.m, a.vScale, 0)
    with pytest.raises(_lib.FbfcError):
        b.loadState(a.m, a.v, a.mScale, a.vScale, -1)


@pytest.mark.gpu
def test_values_without_number_stay_where_they_are():
    """32 bits: an element whose gradient is no number is the only one that changes so.  8 bits: its block of 256 states is."""
    from fbcunn_amd import optim
    for bits in (32, 8):
        (pf, params), (gf, grads) = _tensors([700], "f32", "f32", False, 6)
        grads[0][300], grads[0][301] = float("nan"), float("inf")
        opt = optim.AdamW(params, grads, stateBits=bits, **HYPER)
        opt.step()
        bad = torch.zeros(700, dtype=torch.bool, device="cuda")
        bad[300:302] = True
        assert torch.equal(~params[0].isfinite(), bad)
        if bits == 8:
            assert torch.equal(~opt.mScale.isfinite(), torch.tensor([False, True, False], device="cuda"))
        grads[0].fill_(0.01)
        opt.step()
        if bits == 8:
            bad[256:512] = True
        assert torch.equal(~params[0].isfinite(), bad)


@pytest.mark.gpu
def test_zero_tiny_and_huge_gradients_in_8_bits():
    """A zero block stays zero, values below 2^-100 become zero, and a small positive v beside a large one is never zero."""
    from fbcunn_amd import optim
    (pf, params), (gf, grads) = _tensors([1024], "f32", "f32", False, 6)
    g = grads[0]
    g.zero_()
    g[256:512] = 1e-20            # v = 1e-40 (1 - beta2): below 2^-100, as is not m
    g[512:768] = 1e-4
    g[512] = 1e4
    g[768:] = 1e15
    opt = optim.AdamW(params, grads, stateBits=8, seed=5, **HYPER)
    plain = Plain(opt, 5)
    plain.step(opt.step)
    codes = opt.v.cpu().view(torch.uint8)
    assert int(codes[:512].max()) == 0 and int(codes[512:].min()) >= 1
    assert float(opt.mScale[0]) == 0.0 and float(opt.vScale[1]) == 0.0
    plain.step(opt.step)


@pytest.mark.gpu
def test_rounding_is_unbiased():
    """4096 equal values between two e4m3 neighbours: their mean is theirs to 5 standard deviations of a mean of
    4096 numbers that are a spacing apart (at most 0.5 / 64 of it each)."""
    from fbcunn_amd import optim
    p = torch.zeros(8192, device="cuda")
    g = torch.full((8192,), 0.37, device="cuda")
    g[::256] = 1.0
    opt = optim.AdamW([p], [g], stateBits=8, seed=1, **HYPER)
    opt.step()
    for codes, scales, value, top in ((opt.m, opt.mScale, 0.37 * (1 - 0.9), 1 - 0.9), (opt.v, opt.vScale, 0.37 ** 2 * (1 - 0.95), 1 - 0.95)):
        got = _value(codes, scales).view(-1, 256)[:, 1:].double()
        unit = top / 448
        gap = 2.0 ** (math.floor(math.log2(value / unit)) - 3) * unit
        assert len(got.unique()) == 2
        assert abs(float(got.mean()) - value) <= 5 * 0.5 / math.sqrt(got.numel()) * gap


@pytest.mark.gpu
def test_module_refusals_and_modules():
    from fbcunn_amd import nn, optim
    p, g = torch.zeros(8, device="cuda"), torch.zeros(8, device="cuda")
    for params, grads, error in (([p], [g, g], ValueError), ([p], [g[:4]], ValueError), ([p], [g.double()], TypeError),
                                 ([p[::2]], [g[::2]], ValueError), ([p, p], [g, g], _lib.FbfcError), ([p, p.half()], [g, g], TypeError)):
        with pytest.raises(error):
            optim.AdamW(params, grads)
    with pytest.raises(ValueError):
        optim.AdamW([p], [g], stateBits=4)
    with pytest.raises(_lib.FbfcError):
        optim.AdamW([p], [g], lr=float("nan")).step()
    net = nn.SpatialConvolutionFBFFT(3, 5, 3, 3, 1, 1, 1, 1)
    opt = optim.AdamW.fromModules([net], **HYPER)
    assert opt.params[0] is net.weight and opt.grads[1] is net.gradBias
    x = torch.randn(2, 3, 13, 13, device="cuda")
    net.updateOutput(x)
    net.accGradParameters(x, torch.randn(2, 5, 13, 13, device="cuda"))
    Plain(opt).step(opt.step)


@pytest.mark.gpu
def test_more_than_32_bits_of_parameters():
    """2.2 thousand million parameters in one tensor: its end steps as a tensor of its own does, in both forms of states."""
    from fbcunn_amd import optim
    n, cut = (1 << 31) + (1 << 27) + 77, (1 << 31) + (1 << 27) - 2048     # the cut is a whole block
    gen = torch.Generator("cuda").manual_seed(1)
    p, g = (torch.empty(n, dtype=torch.bfloat16, device="cuda").normal_(generator=gen) for _ in range(2))
    q, h = p[cut:].clone(), g[cut:].clone()
    opt, part = optim.AdamW([p], [g], **HYPER), optim.AdamW([q], [h], **HYPER)
    opt.step(), part.step()
    assert torch.equal(p[cut:], q) and torch.equal(opt.v[cut:], part.v)
    del opt, part
    opt = optim.AdamW([p], [g], stateBits=8, **HYPER)
    before = p[cut:].float()
    opt.step()
    value = opt.m[cut:].float().view(-1, 256) * opt.mScale[cut // 256:, None]
    want = torch.nn.functional.pad(h.float() * (1 - 0.9), (0, -h.numel() % 256)).view(-1, 256)
    assert bool(((value - want).abs() <= 2.0 ** -3 * want.abs() + opt.mScale[cut // 256:, None] * 2.0 ** -9).all())   # one spacing
    assert not torch.equal(p[cut:].float(), before)
    assert len(opt.m[cut:].view(torch.uint8).unique()) > 100


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_states_that_are_refused_change_nothing(bits):
    from fbcunn_amd import optim
    (pf, params), (_, grads) = _tensors([300, 4097], "f32", "f32", False, 8)
    a, b = (optim.AdamW(params, grads, stateBits=bits, **HYPER) for _ in range(2))
    a.step(), b.step(), b.step()
    mine = [t for t in (b.m, b.v, b.mScale, b.vScale) if t is not None]
    before = [t.view(torch.uint8).clone() for t in mine]
    for v, t, error in ((a.v, -1, _lib.FbfcError), (a.v[:256], 1, ValueError), ([0.0], 1, TypeError)):
        with pytest.raises(error):
            b.loadState(a.m, v, a.mScale, a.vScale, t)
        assert all(torch.equal(x.view(torch.uint8), y) for x, y in zip(mine, before)) and b.t == 2


def test_empty_tensors_alone_need_no_states():
    # refused for want of a GPU at most: without parameters there are no elements of states
    for bits in (32, 8):
        rc, message = _create_or_destroy(_config(state_bits=bits), [(0, 0, 0), (0x1000, 0, 0)], m=0, v=0, ms=0, vs=0)
        assert rc in (_lib.OK, _lib.ERR_HIP), message
        rc, message = _create(_config(state_bits=bits), [(0, 0, 0), (0x1000, 0x2000, 1)], m=0, v=0, ms=0, vs=0)
        assert rc == _lib.ERR_INVALID_ARGUMENT and "null" in message


def _create_or_destroy(config, tensors, m, v, ms, vs):
    table = (_lib.AdamwTensor * len(tensors))(*tensors)
    h = ctypes.c_void_p(0)
    rc = _lib.lib().fbfc_adamw_create(ctypes.byref(config), table, len(tensors), m, v, ms, vs, ctypes.byref(h))
    assert bool(h.value) == (rc == _lib.OK)
    message = _lib.lib().fbfc_last_error().decode()
    _lib.lib().fbfc_adamw_destroy(h)
    return rc, message


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_steps_of_empty_tensors_are_counted(bits):
    from fbcunn_amd import optim
    opt = optim.AdamW([torch.zeros(0, 3, device="cuda")], [torch.zeros(0, 3, device="cuda")], stateBits=bits, **HYPER)
    opt.step(), opt.step()
    assert opt.t == 2 and opt.m.numel() == 0
    opt.loadState(opt.m, opt.v, opt.mScale, opt.vScale, 7)
    opt.step()
    assert opt.t == 8
