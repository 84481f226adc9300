"""Preference and policy tuning of a decoder with normed heads and scaled rotations through the runtimes: stages cut
by the planner on CPU devices, and mixed precision with registered weights, eager and under CUDA graphs, on one
GPU, against plain training of the same model."""
import copy
import os

import pytest
import torch

from pfeife_b200 import ops
from pfeife_b200.loss import LossWrapper
from pfeife_b200.models.llama import Llama, llama_config
from pfeife_b200.option import PipeOption


def _model(**overrides):
    torch.manual_seed(0)
    cfg = llama_config("llama_tiny", qk_norm=True, rope_dim=8, rope_interleaved=True,
                       rope_scaling=ops.RopeScaling("bands", 2.0, 16), **overrides)
    model = Llama(cfg)
    with torch.no_grad():
        for name, p in model.named_parameters():
            if name.endswith("norm"):
                p.add_(0.2 * torch.randn_like(p))
    return model


def _batch(n, T, g):
    """Token ids and the labels of their rows: the next token behind a prompt."""
    ids = torch.randint(0, 256, (n, T), generator=g)
    labels = torch.cat([ids[:, 1:], ids.new_full((n, 1), -100)], 1)
    labels[:, :3] = -100
    labels[::2, T - 4:] = -100
    return ids, labels


class PairLoss(LossWrapper):
    def forward(self, input, target, model=None):
        return ops.preference_loss(input, target, input.new_zeros(len(target)), beta=0.05).loss


def test_stages_on_the_cpu():
    from pfeife_b200.runtime.manager import LocalPipeManager
    torch._dynamo.reset()
    model = _model()
    ref = copy.deepcopy(model)
    option = PipeOption(device_cnt=2, batch_size=4, batch_cnt=2, cpu_test=True, no_bench_optimizer=True,
                        verbosity="warning", ctrl_timeout=60, optimizer={"type": "sgd", "lr": 0.05})
    mgr = LocalPipeManager(model, PairLoss(), option)
    ropt = torch.optim.SGD(ref.parameters(), lr=0.05)
    g = torch.Generator().manual_seed(1)
    try:
        for _ in range(2):
            ids, labels = _batch(8, 16, g)
            losses = mgr.run(labels, ids)
            ropt.zero_grad()
            want = []
            for i, l in zip(ids.chunk(2), labels.chunk(2)):
                loss = PairLoss()(ref(i), l)
                loss.backward()
                want.append(float(loss.detach()))
            ropt.step()
            assert [float(l) for l in losses] == pytest.approx(want, abs=1e-5)
        mgr.gather_params()
        for p, q in zip(model.parameters(), ref.parameters()):
            assert torch.allclose(p, q, atol=1e-5)
    finally:
        mgr.close()


@pytest.mark.gpu
@pytest.mark.parametrize("cuda_graphs", [False, True])
def test_mixed_precision_on_one_gpu(cuda_graphs):
    os.environ.setdefault("WORLD_SIZE", "1")
    os.environ.setdefault("RANK", "0")
    os.environ.setdefault("MASTER_PORT", "29879")
    from pfeife_b200 import PartialRunner, initialize_pfeife, partial_compiler
    from pfeife_b200.ops import kernels as kx
    dev = initialize_pfeife().device
    model = _model(num_layers=2).to(dev)
    ref = copy.deepcopy(model)
    opt, ropt = (torch.optim.SGD(m.parameters(), lr=0.1) for m in (model, ref))
    option = PipeOption(device_cnt=1, batch_size=4, batch_cnt=2, mixed_precision="bf16", no_bench_optimizer=True,
                        cuda_graphs=cuda_graphs, verbosity="warning")
    runner = PartialRunner(option, opt)
    torch._dynamo.reset()
    cm = torch.compile(model, backend=partial_compiler)

    def objective(logits, labels, old):
        return ops.policy_loss(logits, labels, old, old[:, :1] + 6.0, old, clip_low=1.0, clip_high=5.0,
                               kl_coef=0.1).loss

    def fn(ids, labels, old):
        loss = objective(cm(ids), labels, old)
        runner.scaler.scale(loss).backward()
        return loss.detach()

    runner.set_exec_fn(fn)
    g = torch.Generator().manual_seed(3)
    start = [p.detach().clone() for p in ref.parameters()]
    for _ in range(4):
        ids, labels = (t.to(dev) for t in _batch(8, 16, g))
        old = torch.full((8, 16), -5.5, device=dev)
        out = runner.step(ids, labels, old)
        ropt.zero_grad()
        for i, (a, b, c) in enumerate(zip(ids.chunk(2), labels.chunk(2), old.chunk(2))):
            loss = objective(ref(a), b, c)
            loss.backward()
            # rows of 256 logits of some 0.1, each rounded to 8 bits several times
            assert float(out[i]) == pytest.approx(float(loss.detach()), rel=3e-2, abs=3e-2)
        ropt.step()
    torch.cuda.synchronize()
    kx.check_status()
    runner.gather_params()
    graphs = len(runner.worker.graphs)
    runner.close()
    ops.unregister_params()              # later calls of this process are of plain tensors again
    assert (graphs > 0) == cuda_graphs
    for (name, p), q, s in zip(model.named_parameters(), ref.parameters(), start):
        # the way that a weight went: some 40 roundings of 2^-9 lie between it and its gradient, four steps
        moved = (q.detach() - s).norm()
        assert float((p.detach().float() - q.detach()).norm()) <= 0.1 * float(moved) + 1e-6, name
        assert moved > 0
