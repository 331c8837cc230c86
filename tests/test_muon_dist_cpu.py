"""FusedMuon behind the bucketed reducer, gloo, two and four ranks: this file is the test and, started by
``torch.distributed.run``, its worker."""
import os
import subprocess
import sys

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)


@pytest.mark.parametrize("world", [2, 4])
def test_fused_muon_data_parallel_gloo(tmp_path, world):
    env = dict(os.environ, OMP_NUM_THREADS="2", DTP_PG_TIMEOUT_S="60")
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=%d" % world, "--master-addr",
           "127.0.0.1", "--master-port", str(29900 + os.getpid() % 90 + world), os.path.abspath(__file__), str(tmp_path)]
    r = subprocess.run(cmd, cwd=ROOT, env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-4000:]
    assert sorted(os.listdir(tmp_path)) == ["ok.%d" % i for i in range(world)]


def _worker(out):
    """Every rank its own images.  After each step all ranks hold the same bits, and those of a model by itself that is
    given the averaged gradient; the reducer refuses to shard the optimizer or to run it per bucket."""
    import torch.distributed as dist
    from distributed_training_pytorch_amd.models import FusedModel
    from distributed_training_pytorch_amd.ops.layers import GroupNormAct
    from distributed_training_pytorch_amd.ops.optim import FusedMuon
    from distributed_training_pytorch_amd.parallel import comm, env as penv
    from distributed_training_pytorch_amd.parallel.data_parallel import DataParallel

    class Net(FusedModel):
        def __init__(self):
            super().__init__()
            self.c = nn.Conv2d(3, 8, 3, padding=1)
            self.n = GroupNormAct(2, 8)
            self.a = nn.Linear(8, 40)
            self.b = nn.Linear(40, 24)
            self.head = nn.Linear(24, 3)
            self.finalize()

        def forward(self, x):
            x = self.n(self.c(x)).mean((2, 3))
            return self.head(F.relu(self.b(F.relu(self.a(x)))))

    penv.ddp_setup("gloo", timeout_s=60)
    rank = dist.get_rank()
    torch.manual_seed(3 + rank)
    net, twin = Net(), Net()
    dp = DataParallel(net, bucket_cap_mb=0.002, first_bucket_mb=0.001)
    twin.load_state_dict(net.state_dict())
    opt, topt = FusedMuon(net, lr=0.01), FusedMuon(twin, lr=0.01)
    for how in ("shard_optimizer", "bucket_optimizer"):
        other = Net()
        with pytest.raises(ValueError, match="neither sharded"):
            DataParallel(other, **{how: FusedMuon(other, lr=0.01)})
    g = torch.Generator().manual_seed(50 + rank)
    for it in range(3):
        x, y = torch.randn(4, 3, 6, 6, generator=g), torch.randint(0, 3, (4,), generator=g)
        opt.zero_grad()
        F.cross_entropy(dp(x), y).backward()
        topt.zero_grad()
        for p, q in zip(net.parameters(), twin.parameters()):
            q.grad.copy_(p.grad)
        opt.step()
        topt.step()
        flat = net.param_arena.flat_master
        assert torch.equal(flat, twin.param_arena.flat_master), it
        lo, hi = flat.clone(), flat.clone()
        dist.all_reduce(lo, op=dist.ReduceOp.MIN)
        dist.all_reduce(hi, op=dist.ReduceOp.MAX)
        assert torch.equal(lo, hi), it
    comm.barrier()
    open(os.path.join(out, "ok.%d" % rank), "w").write("ok")
    penv.destroy_process()


if __name__ == "__main__":
    _worker(sys.argv[1])
