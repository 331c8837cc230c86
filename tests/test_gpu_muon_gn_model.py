"""VGG16 with GroupNorm trained by FusedMuon on the GPU: the operators together, as they are used."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _parts(grad_dtype=F32, dropout=0.3, seed=0, size=64, batch=4, **opt):
    from distributed_training_pytorch_amd.models import vgg16_gn
    from distributed_training_pytorch_amd.ops.layers import SoftmaxCrossEntropy
    from distributed_training_pytorch_amd.ops.optim import FusedMuon
    torch.manual_seed(seed)
    model = vgg16_gn(3, 5, groups=32, dropout=dropout, grad_dtype=grad_dtype).cuda().train()
    x = torch.randn(batch, 3, size, size, device="cuda")
    y = torch.randint(0, 5, (batch,), device="cuda")
    return model, FusedMuon(model, lr=1e-3, **opt), SoftmaxCrossEntropy(), x, y


def _step(model, opt, crit, x, y):
    opt.zero_grad()
    loss = crit(model(x), y)
    loss.backward()
    opt.step()
    return loss.detach()


def _least_cosine(name):
    """What signs and arg-maxes alone may cost a gradient.  Activations are stored in bf16: behind layer j they are off
    by at most e = j * 2^-8 of their size.  A ReLU decides otherwise than in f32 where |z| < e: of values of unit
    spread, a share of 2 * 0.4 * e; each such place carries (or loses) a whole gradient value, so the squared relative
    error of everything below it grows by 0.8 e.  A max-pool decides otherwise where its two largest values are that
    near: the same share.  With S the sum over the layers at and above a parameter, cos >= 1 / sqrt(1 + S); 0.01 for the
    smooth roundings (16 * 2^-8 of either way: 1 - (2 * 0.0625)^2 / 2)."""
    convs = (2, 2, 3, 3, 3)
    layer, last = 0, []                                  # index of every block's last layer: the pool's
    for n in convs:
        layer += n
        last.append(layer)
    if name.startswith("backbone"):
        block, idx = int(name.split(".")[1]), int(name.split(".")[3])
        mine = last[block] - convs[block] + idx // 3 + 1
    else:
        mine = {"linear1": 14, "linear2": 15, "linear3": 16}[name.split(".")[0]]
    s = sum(0.8 * j / 256 for j in range(mine, 16)) + sum(0.8 * j / 256 for j in last if j >= mine)
    return (1 + s) ** -0.5 - 0.01


def test_vgg16_gn_forward_and_gradients_against_cpu():
    """Logits: sixteen layers of bf16 storage, each a rounding of at most 2^-8: 6 % (2-norm)."""
    from distributed_training_pytorch_amd.models import vgg16_gn
    model, opt, crit, x, y = _parts(dropout=0.0)
    cpu = vgg16_gn(3, 5, groups=32, dropout=0.0).train()
    cpu.load_state_dict({k: v.cpu() for k, v in model.state_dict().items()})
    opt.zero_grad()
    logits = model(x)
    crit(logits, y).backward()
    ref = cpu(x.cpu())
    torch.nn.functional.cross_entropy(ref, y.cpu()).backward()
    assert (logits.detach().cpu() - ref.detach()).norm() <= 0.0625 * ref.detach().norm()
    a = model.param_arena
    for (n, p), q in zip(model.named_parameters(), cpu.parameters()):
        g, r = a._logical_view(a.flat_grad, a.index[id(p)]).cpu().flatten().double(), q.grad.flatten().double()
        cos = (g @ r / (g.norm() * r.norm()).clamp_min(1e-30)).item()
        assert cos >= _least_cosine(n), (n, cos, _least_cosine(n))


def test_vgg16_gn_is_the_same_in_eval_mode_and_image_by_image():
    model, _, _, x, _ = _parts(dropout=0.0)
    with torch.no_grad():
        a = model(x)
        model.eval()
        b = model(x)
        c = torch.cat([model(x[i:i + 1].contiguous()) for i in range(4)])
    assert torch.equal(a, b)
    assert torch.allclose(b, c, rtol=0, atol=0.0625 * b.abs().max().item())       # other tiles, other bf16 roundings


@pytest.mark.parametrize("grad_dtype", [F32, BF16])
def test_fused_muon_gpu_matches_cpu(grad_dtype):
    """The same gradients through the GPU's kernels and the CPU's f32 loop.  Both are within 2e-4 of the exact
    orthogonalised direction (2-norm) and round w a few times a step."""
    from distributed_training_pytorch_amd.models import vgg16_gn
    from distributed_training_pytorch_amd.ops.optim import FusedMuon
    model, opt, _, _, _ = _parts(grad_dtype)
    cpu = vgg16_gn(3, 5, groups=32, grad_dtype=F32)
    cpu.load_state_dict({k: v.cpu() for k, v in model.state_dict().items()})
    keep = ("backbone.0.", "backbone.1.", "backbone.2.conv.0", "linear3.")       # (the large matrices take the CPU minutes)
    big = lambda n, p: p.dim() >= 2 and n.startswith(keep[:3])                    # noqa: E731
    opt = FusedMuon(model, lr=1e-2, use_muon=big)
    oc = FusedMuon(cpu, lr=1e-2, use_muon=big)
    a, b = model.param_arena, cpu.param_arena
    before = a.flat_master.clone()
    for t in range(3):
        g = torch.Generator().manual_seed(t)
        grads = (1e-3 * torch.randn(a.total, generator=g)).to(grad_dtype)
        for i, p in enumerate(a.params):                 # padding of the arena stays zero
            o, n = a.offsets[i], p.numel()
            a.flat_grad[o:o + n].copy_(grads[o:o + n])
            b.flat_grad[o:o + n].copy_(grads[o:o + n].float())
        a.fresh = [False] * len(a.params)
        opt.step()
        oc.step()
    for i, n in enumerate(a.names):
        o, k = a.offsets[i], a.params[i].numel()
        x, y, w0 = a.flat_master[o:o + k].cpu().double(), b.flat_master[o:o + k].double(), before[o:o + k].cpu().double()
        assert (x - y).norm() <= 3 * (4e-4 * (y - w0).norm() + 2.0 ** -22 * y.norm()), n
        assert torch.equal(a.flat_lp[o:o + k], a.flat_master[o:o + k].to(BF16)), n
    assert torch.equal(a.flat_master[a.total:], before[a.total:])


@pytest.mark.parametrize("grad_dtype", [F32, BF16])
def test_training_runs_and_repeats_bit_for_bit(grad_dtype):
    runs = []
    for _ in range(2):
        model, opt, crit, x, y = _parts(grad_dtype)
        losses = [float(_step(model, opt, crit, x, y)) for _ in range(4)]
        assert all(v == v for v in losses)
        runs.append((losses, model.param_arena.flat_master.clone()))
    assert runs[0][0] == runs[1][0] and torch.equal(runs[0][1], runs[1][1])


def test_captured_step_equals_eager_step():
    from distributed_training_pytorch_amd.engine.graph import GraphedTrainStep
    model, opt, crit, x, y = _parts(dropout=0.0)
    eager = [float(_step(model, opt, crit, x, y)) for _ in range(7)]
    want = model.param_arena.flat_master.clone()
    model, opt, crit, x, y = _parts(dropout=0.0)
    g = GraphedTrainStep(model, crit, opt, warmup=2)
    assert g.enabled
    got = []
    for k in range(7):
        got.append(float(g(x, y)))
        if k == 4:                                       # the program's own eager work between two replays
            with torch.no_grad():
                model(x)
            torch.cuda.synchronize()
    assert g.replays == 5 and g.captures == 1
    assert got == eager and torch.equal(model.param_arena.flat_master, want)
    assert opt._steps == 7 and int(opt._step_device) == 7


def test_a_graph_of_the_callers_own_counts_its_steps():
    """optimizer.step() alone in a graph: each replay equals an eager step with the same gradients, and the snapshot
    holds the number of steps that ran."""
    model, opt, crit, x, y = _parts(dropout=0.0)
    _step(model, opt, crit, x, y)
    ref, ropt, _, _, _ = _parts(dropout=0.0)
    ref.load_state_dict(copy.deepcopy(model.state_dict()))
    ropt.load_state_dict(copy.deepcopy(opt.state_dict()))
    ropt.zero_grad()
    crit(ref(x), y).backward()
    opt.zero_grad()
    crit(model(x), y).backward()
    assert torch.equal(model.param_arena.flat_grad, ref.param_arena.flat_grad)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opt.step()
    for k in range(3):
        g.replay()
        ropt.step()
        torch.cuda.synchronize()
        assert torch.equal(model.param_arena.flat_master, ref.param_arena.flat_master), k
    assert opt.state_dict()["fused_steps"] == ropt.state_dict()["fused_steps"] == 4


def test_resume_continues_bit_for_bit():
    model, opt, crit, x, y = _parts(dropout=0.0)
    for _ in range(2):
        _step(model, opt, crit, x, y)
    msd, osd = copy.deepcopy(model.state_dict()), copy.deepcopy(opt.state_dict())
    for _ in range(2):
        _step(model, opt, crit, x, y)
    other, o2, crit, x, y = _parts(dropout=0.0)
    other.load_state_dict(msd)
    o2.load_state_dict(osd)
    for _ in range(2):
        _step(other, o2, crit, x, y)
    assert torch.equal(other.param_arena.flat_master, model.param_arena.flat_master)


def test_layer_takes_gradient_accumulation_and_two_uses_of_its_input():
    """A GroupNormAct inside an arena model: gradients add up over two backward passes, and an input with a second
    consumer gets the sum of both gradients."""
    import torch.nn.functional as F
    from distributed_training_pytorch_amd.models import FusedModel
    from distributed_training_pytorch_amd.ops.layers import GroupNormAct

    class Net(FusedModel):
        def __init__(self):
            super().__init__()
            self.n = GroupNormAct(4, 32, act="silu")
            self.finalize()

        def forward(self, x):
            return self.n(self.prepare_input(x)) + x

    net = Net().cuda().train()
    x = torch.randn(2, 6, 5, 32, device="cuda", requires_grad=True)
    ref = x.detach().double().permute(0, 3, 1, 2).requires_grad_()
    w, b = torch.ones(32, dtype=torch.float64, device="cuda", requires_grad=True), torch.zeros(32, dtype=torch.float64, device="cuda", requires_grad=True)
    for _ in range(2):
        (net(x) ** 2).sum().backward()
        ((F.silu(F.group_norm(ref, 4, w, b, 1e-5)) + ref) ** 2).sum().backward()
    a = net.param_arena
    tol = 2.0 ** -24 * 64 * 8                            # 60 values a channel, a few operations each, magnitudes below 8
    assert (x.grad.double() - ref.grad.permute(0, 2, 3, 1)).abs().max() <= tol * ref.grad.abs().max()
    for p, r in ((net.n.weight, w), (net.n.bias, b)):
        assert (a.grad(p).double() - r.grad).abs().max() <= tol * r.grad.abs().max()
