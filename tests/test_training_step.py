"""The operators together, as a training step has them: an FFT convolution along the sequence makes the recurrence's input, its
gate and the block's gate; the recurrence's output goes through the norms with gate and residual; AdamW steps all
parameters.  Gradients against automatic differentiation of the whole chain in 64 bits; the step replayed from a graph."""
import pytest
import torch

pytestmark = pytest.mark.gpu

B, C, T, K = 3, 20, 90, 5


class Block:
    def __init__(self, seed, bits=32):
        from fbcunn_amd import nn, optim
        gen = torch.Generator("cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=gen, device="cuda")   # noqa: E731
        self.conv = nn.SpatialConvolutionFBFFT(C, 3 * C, 1, K, 1, 1, 0, K // 2)
        self.conv.weight.copy_(r(3 * C, C, K, 1) * 0.1)
        self.conv.bias.copy_(r(3 * C) * 0.1)
        self.rec, self.norm = nn.GatedLinearRecurrence(C), nn.GatedResidualNorm(C)
        self.rec.bias.copy_(r(C).abs() + 1)
        for p in self.norm.parameters()[0]:
            p.mul_(1 + 0.2 * r(C))
        self.modules = [self.conv, self.rec, self.norm]
        self.opt = optim.AdamW.fromModules(self.modules, lr=1e-3, stateBits=bits, seed=3)
        self.x, self.gr, self.gn = r(B, C, T, 1), r(B, T, C), r(B, T, C)
        self.grad = torch.empty(B, 3 * C, T, 1, device="cuda")
        self.conv.prepareBackward(self.x)

    def step(self):
        planes = self.conv.updateOutput(self.x)
        # channels are planes here: steps lie side by side, and the recurrence takes them as they are
        x, gate, out_gate = (planes[:, i * C:(i + 1) * C, :, 0].transpose(1, 2) for i in range(3))
        y = self.rec.updateOutput([x, gate])
        residual = self.x[..., 0].transpose(1, 2).contiguous()
        inputs = [residual, y, out_gate.contiguous()]
        self.norm.updateOutput(inputs)
        _, gy, gz = self.norm.backward(inputs, [self.gr, self.gn])
        gx, gg = self.rec.backward([x, gate], gy)
        for i, g in enumerate((gx, gg, gz)):
            self.grad[:, i * C:(i + 1) * C, :, 0].copy_(g.transpose(1, 2))
        self.conv.backward(self.x, self.grad)
        self.opt.step()

    def parameters(self):
        return [p for m in self.modules for p in m.parameters()[0]]

    def gradients(self):
        return [g for m in self.modules for g in m.parameters()[1]]


def _plain(block):
    """The gradients of the parameters, before a step."""
    p = [t.detach().cpu().double().requires_grad_(True) for t in block.parameters()]
    weight, bias, rbias, post, scale, pre = p
    x = block.x.cpu().double()
    planes = torch.nn.functional.conv2d(x, weight, bias, padding=(K // 2, 0))[..., 0].transpose(1, 2)
    v, gate, out_gate = planes.split(C, 2)
    a, h, ys = torch.sigmoid(gate + rbias), torch.zeros(B, C, dtype=torch.float64), []
    for t in range(T):
        h = a[:, t] * h + (1 - a[:, t]) * v[:, t]
        ys.append(h)
    y = torch.stack(ys, 1)
    rms = lambda t: (t.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()   # noqa: E731
    out = x[..., 0].transpose(1, 2) + scale * torch.sigmoid(out_gate) * post * y / rms(y)
    normed = pre * out / rms(out)
    ((out * block.gr.cpu().double()).sum() + (normed * block.gn.cpu().double()).sum()).backward()
    return [t.grad for t in p]


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_of_the_chain_and_the_step(bits):
    block = Block(1, bits)
    for _ in range(3):
        want, before = _plain(block), [p.clone() for p in block.parameters()]
        block.step()
        torch.cuda.synchronize()
        # relative L2 2e-5, the convolution's own bound against the direct form; what follows it rounds at 6e-8 a step
        for got, w in zip(block.gradients(), want):
            assert float((got.cpu().double() - w).norm() / w.norm()) <= 2e-5
        for p, old in zip(block.parameters(), before):
            moved = (p - old).abs()
            assert float(moved.max()) <= 1.2e-3 * 3.2 and float(moved.mean()) > 1e-4   # of the order of lr


@pytest.mark.parametrize("bits", [32, 8])
def test_the_step_replays_from_a_graph(bits):
    block, eager = Block(2, bits), Block(2, bits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            block.step()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block.step()
    for rep in range(4):
        for g in block.gradients():
            g.fill_(float("nan"))
        block.x.mul_(-0.9), eager.x.mul_(-0.9)
        (block.x * 2).sum().item()
        graph.replay()
        torch.cuda.synchronize()
        eager.step()
        for a, b in zip(block.parameters() + block.gradients(), eager.parameters() + eager.gradients()):
            assert torch.equal(a, b), rep
    assert block.opt.t == eager.opt.t == 6
