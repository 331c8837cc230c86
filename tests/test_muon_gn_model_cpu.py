"""FusedMuon and GroupNormAct on the CPU: the update rule in 64 bits, state, refusals, the entry points."""
import math
import os
import subprocess
import sys

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from distributed_training_pytorch_amd.models import FusedModel, VGG16, vgg16_gn
from distributed_training_pytorch_amd.ops.layers import GroupNormAct
from distributed_training_pytorch_amd.ops.optim import FusedMuon

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Tiny(FusedModel):
    def __init__(self):
        super().__init__()
        self.c = nn.Conv2d(3, 8, 3, padding=1)
        self.n = GroupNormAct(2, 8, act="silu")
        self.a = nn.Linear(8, 12)
        self.head = nn.Linear(12, 3)
        self.finalize()

    def forward(self, x):
        return self.head(F.relu(self.a(self.n(self.c(x)).mean((2, 3)))))


def _grads(model, seed):
    g = torch.Generator().manual_seed(seed)
    for p in model.parameters():
        p.grad.copy_(torch.randn(p.shape, generator=g))


def _ns64(x, steps=5, co=(3.4445, -4.7750, 2.0315)):
    x = x / (x.norm() + 1e-7)
    for _ in range(steps):
        u, s, vt = torch.linalg.svd(x, full_matrices=False)       # the polynomial, applied to the singular values
        x = u @ torch.diag(co[0] * s + co[1] * s ** 3 + co[2] * s ** 5) @ vt
    return x


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("adjust", ["match_rms_adamw", "original"])
def test_fused_muon_cpu_rule(nesterov, adjust):
    torch.manual_seed(0)
    m = Tiny()
    opt = FusedMuon(m, lr=0.02, weight_decay=0.1, nesterov=nesterov, adjust_lr=adjust)
    names = m.param_arena.names
    assert [names[i] for i in opt._muon] == ["c.weight", "a.weight"]
    w = {n: p.detach().double().clone() for n, p in m.named_parameters()}
    mom = {n: torch.zeros_like(v) for n, v in w.items()}
    sq = {n: torch.zeros_like(v) for n, v in w.items()}
    for t in range(1, 4):
        _grads(m, t)
        grads = {n: p.grad.double() for n, p in m.named_parameters()}
        opt.step()
        for n in w:
            g = grads[n]
            if n in ("c.weight", "a.weight"):
                mom[n] = 0.95 * mom[n] + 0.05 * g
                u = 0.05 * g + 0.95 * mom[n] if nesterov else mom[n]
                u2 = u.reshape(u.shape[0], -1)
                s = 0.2 * math.sqrt(max(u2.shape)) if adjust == "match_rms_adamw" else math.sqrt(max(1, u2.shape[0] / u2.shape[1]))
                w[n] = w[n] * (1 - 0.02 * 0.1) - 0.02 * s * _ns64(u2).reshape(u.shape)
            else:
                mom[n] = 0.9 * mom[n] + 0.1 * g
                sq[n] = 0.95 * sq[n] + 0.05 * g * g
                w[n] = w[n] * (1 - 0.02 * 0.1) - 0.02 / (1 - 0.9 ** t) * mom[n] / ((sq[n] / (1 - 0.95 ** t)).sqrt() + 1e-8)
    for n, p in m.named_parameters():
        # f32 rounding of three steps; the iteration amplifies a rounding of X by at most a^5 = 484 in directions of no size
        assert (p.detach().double() - w[n]).abs().max() <= 3 * (484 * 2.0 ** -24 * 0.02 * 0.2 * 5.2 + 2.0 ** -22), n


def test_fused_muon_state_roundtrip_and_refusals():
    torch.manual_seed(0)
    a = Tiny()
    oa = FusedMuon(a, lr=0.01)
    for t in range(2):
        _grads(a, t)
        oa.step()
    sd, msd = oa.state_dict(), a.state_dict()
    assert set(sd["state"][0]) == {"momentum_buffer"} and set(sd["state"][1]) == {"momentum_buffer", "exp_avg_sq"}
    b = Tiny()
    ob = FusedMuon(b, lr=0.5)
    b.load_state_dict(msd)
    ob.load_state_dict(sd)
    assert ob.param_groups[0]["lr"] == 0.01 and ob._steps == 2 and int(ob._step_device) == 2
    for t in range(2, 4):
        _grads(a, t)
        _grads(b, t)
        oa.step()
        ob.step()
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q)
    other = FusedMuon(Tiny(), use_muon=lambda n, p: n == "head.weight")
    with pytest.raises(ValueError, match="divides the parameters"):
        other.load_state_dict(sd)
    with pytest.raises(ValueError, match="neither sharded"):
        oa._sharded_by = object()
    oa._sharded_by = None
    assert not hasattr(oa, "update_range")          # the Trainer keeps it out of the per-bucket path
    for kw, what in ((dict(momentum=1.0), "momentum"), (dict(adjust_lr="x"), "adjust_lr"), (dict(betas=(0.9, 1.0)), "betas"),
                     (dict(ns_steps=0), "steps"), (dict(adamw_eps=0.0), "adamw_eps"), (dict(ns_coeffs=(9.0, 9.0, 9.0)), "bounded")):
        with pytest.raises(ValueError, match=what):
            FusedMuon(Tiny(), **kw)


def test_group_norm_act_cpu_and_refusals():
    x = torch.randn(2, 8, 5, 4)
    for act, f in (("none", lambda v: v), ("relu", F.relu), ("silu", F.silu)):
        m = GroupNormAct(4, 8, act=act)
        assert torch.equal(m(x), f(F.group_norm(x, 4, m.weight, m.bias, 1e-5)))
    for g, c, act in ((3, 8, "relu"), (0, 8, "relu"), (2, 8, "gelu")):
        with pytest.raises(ValueError):
            GroupNormAct(g, c, act=act)
    with pytest.raises(ValueError, match="not both"):
        VGG16(3, 2, batch_norm=True, group_norm=32)


def test_vgg16_gn_matches_a_stock_torch_model():
    torch.manual_seed(0)
    m = vgg16_gn(3, 5, groups=32).eval()
    layers, cin = [], 3
    for c, n in ((64, 2), (128, 2), (256, 3), (512, 3), (512, 3)):
        block = []
        for _ in range(n):
            block += [nn.Conv2d(cin, c, 3, padding=1), nn.GroupNorm(32, c), nn.ReLU()]
            cin = c
        layers.append(nn.ModuleDict({"conv": nn.Sequential(*block, nn.MaxPool2d(2, 2))}))
    stock = nn.Module()
    stock.backbone = nn.Sequential(*layers)
    stock.linear1, stock.linear2, stock.linear3 = nn.Linear(25088, 4096), nn.Linear(4096, 4096), nn.Linear(4096, 5)
    stock.load_state_dict(m.state_dict(), strict=True)
    x = torch.randn(2, 3, 32, 32)
    with torch.no_grad():
        y = x
        for b in stock.backbone:
            y = b["conv"](y)
        y = torch.flatten(F.adaptive_avg_pool2d(y, (7, 7)), 1)
        y = stock.linear3(F.relu(stock.linear2(F.relu(stock.linear1(y)))))
        assert torch.allclose(m(x), y, rtol=1e-4, atol=1e-5)


def test_main_runs_with_group_norm_and_muon(tmp_path):
    cmd = [sys.executable, "main.py", "--synthetic", "--synthetic-size", "4", "--epochs", "1", "--batch-size", "2",
           "--image-size", "32", "--no-progress", "--steps", "1", "--no-validate", "--group-norm", "32", "--optimizer", "muon",
           "--lr", "0.001", "--save-folder", str(tmp_path), "--backend", "gloo"]
    env = dict(os.environ, CUDA_VISIBLE_DEVICES="", HIP_VISIBLE_DEVICES="")
    r = subprocess.run(cmd, cwd=ROOT, env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-3000:]


@pytest.mark.parametrize("given,want", [
    (dict(), (0.1, 0.9)), (dict(lr=0.02, momentum=0.5), (0.02, 0.5)), (dict(optimizer="muon"), (1e-3, 0.95)),
    (dict(optimizer="muon", lr=0.02), (0.02, 0.95)), (dict(optimizer="muon", momentum=0.8), (1e-3, 0.8))])
def test_trainer_gives_each_optimizer_its_own_lr_and_momentum(given, want, monkeypatch):
    """Muon at SGD's lr of 0.1 moves every matrix by a tenth of its size a step; a momentum that is given counts."""
    import main
    from distributed_training_pytorch_amd.trainer.example_trainer import ExampleTrainer
    from distributed_training_pytorch_amd.trainer.trainer import Trainer
    monkeypatch.setattr(Trainer, "__init__", lambda self, *a, **k: None)
    t = ExampleTrainer("train", "val", ["a"], 32, 32, 1, 2, False, **given)
    t.model = Tiny()
    g = t.build_optimizer().param_groups[0]
    assert (g["lr"], g["momentum"]) == want
    assert main.parse_args([]).lr is None
