"""What is measured of the training and serving operators: the gated linear recurrence, the gated residual norm and
the AdamW step.  `run` computes them from elementary torch operations where `own` is false and through
fbcunn_amd where it is true."""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_EPS = 1e-6
# AdamW: hyper-parameters, and the constants of the random numbers that 8-bit states are rounded with
_LR, _B1, _B2, _ADAM_EPS, _DECAY, _SEED, _T0 = 3e-4, 0.9, 0.95, 1e-8, 0.1, 1234, 100
_K1, _K2, _K3 = 0x9E3779B1, 0xBB67AE85, 0xB504F335
_BLOCK = 256


def listed():
    rec = dict(op="recurrence", lengths=False)
    norm = dict(op="norm", form="full")
    return [
        # one token for each of 64 sequences being served
        dict(rec, name="recurrence step", batch=64, steps=1, channels=4096, type="bf16", **{"pass": "step"}),
        # a batch of prompts
        dict(rec, name="recurrence forward", batch=8, steps=2048, channels=1024, type="bf16", **{"pass": "forward"}),
        # a padded batch of sequences of odd sizes, trained in 32 bits
        dict(rec, name="recurrence train ragged", batch=5, steps=1537, channels=515, type="f32", **{"pass": "train", "lengths": True}),
        # one very long sequence, trained
        dict(rec, name="recurrence train long", batch=1, steps=131072, channels=2048, type="bf16", **{"pass": "train"}),
        # the tokens of 16 sequences being served
        dict(norm, name="norm tokens", rows=16, channels=4096, type="bf16", **{"pass": "forward"}),
        # a training batch's forward pass
        dict(norm, name="norm forward", rows=8192, channels=2048, type="bf16", **{"pass": "forward"}),
        # an odd width in 32 bits, backwards
        dict(norm, name="norm backward odd", rows=3001, channels=1000, type="f32", **{"pass": "backward"}),
        # a large training batch backwards
        dict(norm, name="norm backward large", rows=65536, channels=4096, type="bf16", **{"pass": "backward"}),
        # the layers of a small network whose parameters were flattened into one storage
        dict(op="adamw", name="adamw few small", tensors=8, elements=300007, param="f32", grad="f32", bits=32, packed=True),
        # the tensors of a mid-sized network
        dict(op="adamw", name="adamw many", tensors=160, elements=40000000, param="f32", grad="f32", bits=32, packed=False),
        # the same with 8-bit states and parameters of 16 bits, packed without alignment
        dict(op="adamw", name="adamw 8 bit many", tensors=120, elements=25000001, param="bf16", grad="bf16", bits=8, packed=True),
        # a large network: parameters in 32 bits, gradients in 16, states in 8
        dict(op="adamw", name="adamw 8 bit large", tensors=200, elements=250000000, param="f32", grad="bf16", bits=8, packed=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("recurrence", "norm", "adamw"))
    if op == "recurrence":
        way = rng.choice(("step", "forward", "train", "train"))
        channels = _log(rng, 16, 4096)
        steps = 1 if way == "step" else _log(rng, 1, 65536)
        batch = _log(rng, 1, max(1, min(256 if way == "step" else 64, (1 << 27) // (channels * steps))))
        return {"op": op, "pass": way, "batch": batch, "steps": steps, "channels": channels,
                "type": rng.choice(("f32", "bf16", "f16")), "lengths": way != "step" and rng.random() < 0.4}
    if op == "norm":
        channels = _log(rng, 16, 12000)
        return {"op": op, "pass": rng.choice(("forward", "backward")), "rows": _log(rng, 1, min(65536, (1 << 27) // channels)),
                "channels": channels, "type": rng.choice(("f32", "bf16", "f16")),
                "form": rng.choice(("full", "full", "ungated", "last", "first"))}
    tensors = _log(rng, 1, 250)
    param, grad = rng.choice((("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f16")))
    return {"op": op, "tensors": tensors, "elements": _log(rng, max(1000, 4 * tensors), 1 << 27), "param": param, "grad": grad,
            "bits": rng.choice((32, 8)), "packed": rng.random() < 0.5}


def work(case):
    if case["op"] == "recurrence":
        b, t, d, e = case["batch"], case["steps"], case["channels"], _BYTES[case["type"]]
        whole, read = b * t * d, sum(_lengths(case)) * d
        state = 8 * b * d + 4 * d
        if case["pass"] == "train":
            return {"bytes": e * (3 * read + 3 * whole) + 2 * state, "flops": 37 * read}
        return {"bytes": e * (2 * read + whole) + state, "flops": 12 * read}
    if case["op"] == "norm":
        n, d, e = case["rows"] * case["channels"], case["channels"], _BYTES[case["type"]]
        branch, gate, pre = _form(case)
        read = 1 + branch + gate
        if case["pass"] == "forward":
            return {"bytes": e * n * (read + branch + pre) + 4 * d * (2 * branch + pre), "flops": 16 * n}
        return {"bytes": e * n * (read + branch + pre + 1 + branch + gate) + 8 * d * (2 * branch + pre), "flops": 40 * n}
    n = case["elements"]
    state = 16 if case["bits"] == 32 else 4 + 16.0 / _BLOCK
    return {"bytes": n * (2 * _BYTES[case["param"]] + _BYTES[case["grad"]] + state), "flops": (16 if case["bits"] == 32 else 60) * n}


def _generator(seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


# recurrence ---------------------------------------------------------------------------------------------

def _lengths(case):
    """Lengths of a padded batch: from the full one down to a few steps, one of them empty where there are many."""
    b, t = case["batch"], case["steps"]
    if not case["lengths"]:
        return [t] * b
    return [0 if i == b - 1 and b > 3 else t - i * t // b for i in range(b)]


def _prepare_recurrence(case, seed):
    g = _generator(seed)
    b, t, d, dt = case["batch"], case["steps"], case["channels"], _TYPES[case["type"]]
    # decays that last from two steps to some hundreds
    s = {"bias": torch.rand(d, generator=g, device="cuda") * 6, "h0": _normal(g, b, d) * 0.5}
    shape = (b, d) if case["pass"] == "step" else (b, t, d)
    s["x"], s["gate"] = (_normal(g, *shape).to(dt) for _ in range(2))
    if case["pass"] == "train":
        s["gy"], s["gh"] = _normal(g, *shape).to(dt), _normal(g, b, d)
    s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if case["lengths"] else None
    if own:
        from fbcunn_amd import nn
        s["net"] = nn.GatedLinearRecurrence(d)
        s["net"].bias.copy_(s["bias"])
        if case["pass"] == "forward":
            s["net"].evaluate()
    return s


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1, from zero, in a logarithmic number of passes."""
    k = 1
    while k < a.size(1):
        b = torch.cat((b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]), 1)
        a = torch.cat((a[:, :k], a[:, k:] * a[:, :-k]), 1)
        k *= 2
    return b


def _run_recurrence(case, s):
    way = case["pass"]
    if own:
        net = s["net"]
        if way == "step":
            return [net.step([s["x"], s["gate"]], s["h0"]), s["h0"]]
        y = net.updateOutput([s["x"], s["gate"]], state=s["h0"], lengths=s["lengths"])
        if way == "forward":
            return [y, net.state]
        net.backward([s["x"], s["gate"]], s["gy"], gradState=s["gh"])
        if s["gy"].dtype == torch.float32 and s["lengths"] is None:
            # the plain form adds the state's gradient to the last step of these very gradients in place: the next pass on
            # this state has to find them alike
            s["gy"][:, -1] += s["gh"]
        return [y, net.state, net.gradInput[0], net.gradInput[1], net.gradState, net.gradBias]
    dt = s["x"].dtype
    x, z = s["x"].float(), s["gate"].float() + s["bias"]
    a, c = torch.sigmoid(z), torch.sigmoid(-z)
    if way == "step":
        h = a * s["h0"] + c * x
        s["h0"].copy_(h)
        return [h.to(dt), s["h0"]]
    live = None
    if s["lengths"] is not None:
        live = (torch.arange(x.size(1), device=x.device) < s["lengths"][:, None])[..., None]
        x, a, c = torch.where(live, x, 0), torch.where(live, a, 1), torch.where(live, c, 0)
    v = c * x
    v[:, 0] += a[:, 0] * s["h0"]
    h = _scan(a, v)
    y = h if live is None else torch.where(live, h, 0)
    if way == "forward":
        return [y.to(dt), h[:, -1].clone()]
    gy = s["gy"].float() if live is None else torch.where(live, s["gy"].float(), 0)
    gy[:, -1] += s["gh"]
    back = torch.cat((torch.zeros_like(a[:, :1]), a.flip(1)[:, :-1]), 1)
    u = _scan(back, gy.flip(1)).flip(1)
    before = torch.cat((s["h0"][:, None], h[:, :-1]), 1)
    gz = u * (before - x) * a * c
    return [y.to(dt), h[:, -1].clone(), (u * c).to(dt), gz.to(dt), a[:, 0] * u[:, 0], gz.sum((0, 1))]


def _exact_recurrence(case, seed):
    s = _prepare_recurrence(case, seed)
    one = case["pass"] == "step"
    x, z = s["x"].double(), s["gate"].double() + s["bias"].double()
    if one:
        x, z = x[:, None], z[:, None]
    # time first, one step after the other
    x, z = x.transpose(0, 1).contiguous(), z.transpose(0, 1).contiguous()
    a, c = 1 / (1 + torch.exp(-z)), 1 / (1 + torch.exp(z))
    t, dead = x.size(0), None
    if s["lengths"] is not None:
        dead = torch.arange(t, device="cuda")[:, None, None] >= s["lengths"][None, :, None]
        a, c = a.masked_fill(dead, 1), c.masked_fill(dead, 0)
    h = torch.empty_like(x)
    v = c * x
    del z
    last = s["h0"].double()
    for i in range(t):
        last = torch.addcmul(v[i], a[i], last, out=h[i])
    y = (h if dead is None else h.masked_fill(dead, 0)).transpose(0, 1)
    if one:
        return [y[:, 0], last]
    if case["pass"] == "forward":
        return [y, last]
    u = s["gy"].double().transpose(0, 1).contiguous()
    if dead is not None:
        u.masked_fill_(dead, 0)
    u[-1] += s["gh"].double()
    for i in range(t - 2, -1, -1):
        u[i].addcmul_(a[i + 1], u[i + 1])
    gz = torch.cat((s["h0"].double()[None], h[:-1])) - x
    gz *= u * a * c
    return [y, last, (u * c).transpose(0, 1), gz.transpose(0, 1), a[0] * u[0], gz.sum((0, 1))]


# norm ---------------------------------------------------------------------------------------------------

def _form(case):
    """(branch, gate, norm after): which parts of the operator the case has."""
    return {"full": (1, 1, 1), "ungated": (1, 0, 1), "last": (1, 1, 0), "first": (0, 0, 1)}[case["form"]]


def _prepare_norm(case, seed):
    g = _generator(seed)
    n, d, dt = case["rows"], case["channels"], _TYPES[case["type"]]
    branch, gate, pre = _form(case)
    s = {"residual": (_normal(g, n, d) * 2).to(dt), "branch": (_normal(g, n, d) * 0.7).to(dt) if branch else None,
         "gate": _normal(g, n, d).to(dt) if gate else None}
    s["post"], s["scale"], s["pre"] = (1 + 0.2 * _normal(g, d), 0.5 + 0.1 * _normal(g, d), 1 + 0.2 * _normal(g, d))
    if case["pass"] == "backward":
        s["gr"] = _normal(g, n, d).to(dt)
        s["gn"] = _normal(g, n, d).to(dt) if pre else None
    if own:
        from fbcunn_amd import nn
        net = s["net"] = nn.GatedResidualNorm(d, eps=_EPS, branch=bool(branch), gate=bool(gate), norm=bool(pre))
        for mine, given in ((net.postWeight, "post"), (net.scale, "scale"), (net.preWeight, "pre")):
            if mine is not None:
                mine.copy_(s[given])
    return s


def _run_norm(case, s):
    branch, gate, pre = _form(case)
    if own:
        net = s["net"]
        given = [t for t in (s["residual"], s["branch"], s["gate"]) if t is not None]
        if case["pass"] == "forward":
            r, n = net.updateOutput(given)
            return [r if branch else None, n]
        net.backward(given, [s["gr"], s["gn"]])
        return [net.gradInput, net.gradPostWeight, net.gradScale, net.gradPreWeight]
    dt = s["residual"].dtype
    r = s["residual"].float()
    if branch:
        y = s["branch"].float()
        i1 = torch.rsqrt(y.square().mean(1, keepdim=True) + _EPS)
        k = torch.sigmoid(s["gate"].float()) if gate else None
        yn = y * i1
        f = yn * (s["post"] * s["scale"])
        r = r + (k * f if gate else f)
    if pre:
        i2 = torch.rsqrt(r.square().mean(1, keepdim=True) + _EPS)
        rn = r * i2
    if case["pass"] == "forward":
        return [r.to(dt) if branch else None, (rn * s["pre"]).to(dt) if pre else None]
    gr, gpre = s["gr"].float(), None
    if pre:
        gn = s["gn"].float()
        gpre = (gn * rn).sum(0)
        w = gn * s["pre"]
        gr = gr + i2 * (w - rn * (w * rn).mean(1, keepdim=True))
    if not branch:
        return [[gr.to(dt)], None, None, gpre]
    gf = gr * k if gate else gr
    both = (gf * yn).sum(0)
    w = gf * (s["post"] * s["scale"])
    gy = i1 * (w - yn * (w * yn).mean(1, keepdim=True))
    gz = [(gr * f * k * torch.sigmoid(-s["gate"].float())).to(dt)] if gate else []
    return [[gr.to(dt), gy.to(dt)] + gz, both * s["scale"], both * s["post"], gpre]


def _exact_norm(case, seed):
    s = _prepare_norm(case, seed)
    branch, gate, pre = _form(case)
    need = case["pass"] == "backward"
    v = {k: s[k].double().requires_grad_(need) for k in ("residual", "branch", "gate", "post", "scale", "pre") if s[k] is not None}
    r = v["residual"]
    if branch:
        y = v["branch"]
        u = v["post"] * y / (y.pow(2).mean(-1, keepdim=True) + _EPS).sqrt()
        u = v["scale"] * u
        r = r + (u / (1 + torch.exp(-v["gate"])) if gate else u)
    n = v["pre"] * r / (r.pow(2).mean(-1, keepdim=True) + _EPS).sqrt() if pre else None
    if not need:
        return [r if branch else None, n]
    loss = (r * s["gr"].double()).sum()
    if pre:
        loss = loss + (n * s["gn"].double()).sum()
    loss.backward()
    grads = [v[k].grad for k in ("residual", "branch", "gate") if k in v]
    return [grads, v["post"].grad, v["scale"].grad, v["pre"].grad]


# AdamW --------------------------------------------------------------------------------------------------

def _sizes(case):
    """Lengths of the tensors: every other one short, as biases are, the others sharing what is left unevenly."""
    count, left = case["tensors"], case["elements"]
    short = [min(1 + (i * 37) % 1021, max(1, left // (4 * count))) for i in range(1, count, 2)]
    left -= sum(short)
    weight = [1 + (i * i * 7) % 13 for i in range(0, count, 2)]
    long = [max(1, left * w // sum(weight)) for w in weight]
    long[0] += left - sum(long)
    return [long[i // 2] if i % 2 == 0 else short[i // 2] for i in range(count)]


def _prepare_adamw(case, seed):
    g = _generator(seed)
    sizes = _sizes(case)
    pads = [-n % _BLOCK for n in sizes]
    at, total = [], 0
    for n in sizes:
        at.append(total)
        total += n if case["packed"] else -(-n // 64) * 64
    s = {"t": _T0, "sizes": sizes, "pads": pads}
    for name, kind, size in (("param", "param", 0.05), ("grad", "grad", 0.01)):
        s[name + "_all"] = flat = (_normal(g, total) * size).to(_TYPES[case[kind]])
        s[name + "s"] = [flat[o:o + n] for o, n in zip(at, sizes)]
    n = sum(sizes) + sum(pads)
    real = torch.cat([torch.cat((torch.ones(a, device="cuda"), torch.zeros(b, device="cuda"))) for a, b in zip(sizes, pads)])
    m, v = _normal(g, n).mul_(0.004).mul_(real), _normal(g, n).mul_(0.01).square_().add_(1e-6).mul_(real)
    if case["bits"] == 8:
        for name, x in (("m", m), ("v", v)):
            x = x.view(-1, _BLOCK)
            scale = x.abs().amax(1) * (1 / 448)
            s[name] = (x / scale[:, None]).clamp_(-448, 448).to(torch.float8_e4m3fn).view(-1)
            s[name + "_scale"] = scale
    else:
        s["m"], s["v"], s["m_scale"], s["v_scale"] = m, v, None, None
    s["zeros"] = [[torch.zeros(b, dtype=_TYPES[case[kind]], device="cuda") for b in pads] for kind in ("param", "grad")]
    if own:
        from fbcunn_amd import optim
        opt = s["opt"] = optim.AdamW(s["params"], s["grads"], lr=_LR, betas=(_B1, _B2), eps=_ADAM_EPS, weightDecay=_DECAY,
                                     stateBits=case["bits"], seed=_SEED)
        opt.loadState(s["m"], s["v"], s["m_scale"], s["v_scale"], s["t"])
    return s


def _flat(tensors, zeros):
    """The tensors one after the other, each filled up to whole blocks."""
    return torch.cat([x for pair in zip(tensors, zeros) for x in pair]).float()


def _random(n, key):
    """Two streams of 20-bit numbers for the n elements of the states."""
    i = torch.arange(n, device="cuda")
    low = 0xFFFFFFFF
    x = ((i & low) * _K1 + (i >> 32) * _K3 + key) & low
    x ^= x >> 16
    x = (x * _K2) & low
    x ^= x >> 15
    x = (x * _K3) & low
    x ^= x >> 16
    y = (x * _K1) & low
    y ^= y >> 16
    y = (y * _K2) & low
    return (x >> 12).int(), (y >> 12).int()


def _round8(x, random, floor):
    """(values in e4m3, scales): each block of 256 divided by its scale and rounded up or down as `random` says, towards
    the nearer value more often.  The bits of a 32-bit float of 2^-120 times the value hold the 8-bit one on top."""
    x = x.view(-1, _BLOCK)
    top = x.abs().amax(1)
    scale = torch.where(top < 2.0 ** -100, 0.0, top * (1 / 448))
    inverse = torch.where(scale > 0, 1 / scale, 0.0)[:, None]
    bits = (x.abs() * inverse * 2.0 ** -120).view(torch.int32)
    code = ((bits + random.view(-1, _BLOCK)) >> 20).clamp_(max=0x7E)
    if floor:
        code = torch.where((code == 0) & (x > 0) & (inverse > 0), 1, code)
    else:
        code = code | (x < 0).int() << 7
    return code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1), scale


def _run_adamw(case, s):
    s["t"] += 1
    if own:
        s["opt"].step()
        opt = s["opt"]
        return [s["param_all"], opt.m, opt.v, opt.mScale, opt.vScale]
    t, small = s["t"], case["bits"] == 8
    p, g = (_flat(x, zeros) for x, zeros in zip((s["params"], s["grads"]), s["zeros"]))
    m, v = s["m"], s["v"]
    if small:
        m, v = ((s[k].view(-1, _BLOCK).float() * s[k + "_scale"][:, None]).view(-1) for k in ("m", "v"))
    m = m * _B1 + g * (1 - _B1)
    v = v * _B2 + g * g * (1 - _B2)
    d = v.sqrt() * (1 / math.sqrt(1 - _B2 ** t)) + _ADAM_EPS
    p = p * (1 - _LR * _DECAY) - m / d * (_LR / (1 - _B1 ** t))
    pieces = torch.split(p, [n for pair in zip(s["sizes"], s["pads"]) for n in pair])
    torch._foreach_copy_(s["params"], list(pieces[::2]))
    if small:
        r = _random(m.numel(), (_SEED * _K1 + t * _K2) & 0xFFFFFFFF)
        for name, x, random in (("m", m, r[0]), ("v", v, r[1])):
            x, scale = _round8(x, random, name == "v")
            s[name].view(torch.uint8).copy_(x.view(torch.uint8))
            s[name + "_scale"].copy_(scale)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return [s["param_all"], s["m"], s["v"], s["m_scale"], s["v_scale"]]


def _exact_adamw(case, seed):
    s = _prepare_adamw(case, seed)
    t = s["t"] + 1
    out = s["param_all"].double()
    new, first, o = {"m": [], "v": [], "m_scale": [], "v_scale": []}, 0, 0
    total = s["m"].numel()
    r = _random(total, (_SEED * _K1 + t * _K2) & 0xFFFFFFFF) if case["bits"] == 8 else None
    for p, g, n, pad in zip(s["params"], s["grads"], s["sizes"], s["pads"]):
        where = slice(first, first + n + pad)
        first += n + pad
        m, v = s["m"][where].double(), s["v"][where].double()
        if r is not None:
            blocks = slice(where.start // _BLOCK, where.stop // _BLOCK)
            m *= s["m_scale"][blocks].double().repeat_interleave(_BLOCK)
            v *= s["v_scale"][blocks].double().repeat_interleave(_BLOCK)
        g = torch.nn.functional.pad(g.double(), (0, pad))
        m, v = _B1 * m + (1 - _B1) * g, _B2 * v + (1 - _B2) * g * g
        step = (m / (1 - _B1 ** t)) / ((v / (1 - _B2 ** t)).sqrt() + _ADAM_EPS)
        o = p.storage_offset()
        out[o:o + n] = p.double() - _LR * _DECAY * p.double() - _LR * step[:n]
        for name, x, k in (("m", m, 0), ("v", v, 1)):
            if r is None:
                new[name].append(x)
                continue
            scale = x.view(-1, _BLOCK).abs().amax(1) / 448
            y = x.abs() / scale.clamp(min=1e-30).repeat_interleave(_BLOCK)
            # spacing of e4m3 around y: 2^-9 below 2^-6, an eighth of the power of two above
            gap = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
            low = torch.floor(y / gap)
            low = (low + (y / gap - low > 1 - r[k][where].double() / 2 ** 20)) * gap
            low = low.clamp(max=448.0)
            if k:
                low = torch.where((low == 0) & (x > 0), 2.0 ** -9, low)
            new[name].append((low * x.sign()).float())
            new[name + "_scale"].append(scale)
    new = {k: torch.cat(v) if v else None for k, v in new.items()}
    return [out, new["m"], new["v"], new["m_scale"], new["v_scale"]]


# ---------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    s = {"recurrence": _prepare_recurrence, "norm": _prepare_norm, "adamw": _prepare_adamw}[case["op"]](case, seed)
    s["case"] = case
    return s


def run(state):
    case = state["case"]
    return {"recurrence": _run_recurrence, "norm": _run_norm, "adamw": _run_adamw}[case["op"]](case, state)


def exact(case, seed):
    """The operators from their definitions in 64 bits, the recurrence one step after the other, the norm's gradients by
    automatic differentiation, AdamW tensor by tensor."""
    return {"recurrence": _exact_recurrence, "norm": _exact_norm, "adamw": _exact_adamw}[case["op"]](case, seed)
