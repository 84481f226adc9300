"""Preference and policy tuning of a decoder with normed heads and scaled rotations through the runtimes: stages cut
by the planner on CPU devices, and mixed precision with registered weights, eager and under CUDA graphs, on one
GPU, against plain training of the same model."""
import copy
import math
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


# ------------------------------------------------------------------------------ pairs and micro-batches
def _documented(name, **names):
    """The function of that name in the user's guide, over the objects given."""
    import re
    from pathlib import Path
    guide = (Path(__file__).resolve().parent.parent / "README.md").read_text()
    for block in re.findall(r"```python\n(.*?)```", guide, re.S):
        if f"def {name}(" in block:
            scope = {"llama_config": llama_config, **names}
            exec(block, scope)
            return scope[name]
    raise AssertionError(f"no {name} in the guide")


def _pairs(P, T, g):
    """[P, 2, T] ids and labels, [P, 2] log-probabilities that lie around those of some 5.5 nats a token."""
    ids, labels = _batch(2 * P, T, g)
    return ids.view(P, 2, T), labels.view(P, 2, T), torch.randn(P, 2, generator=g) * 4 - 5.5 * T


def _pair_loss(logits, labels, ref):
    """Of each pair, from the definition: logits [P, 2, T, V]"""
    l = torch.log_softmax(logits.double(), -1).gather(-1, labels.clamp(min=0).unsqueeze(-1))[..., 0] * (labels >= 0)
    r = 0.1 * (l.sum(-1) - ref.double())
    return -torch.nn.functional.logsigmoid(r[:, 0] - r[:, 1])


class Unscaled:
    """A runner's loss scale where nothing is scaled."""

    class scaler:
        scale = staticmethod(lambda loss: loss)


@pytest.mark.parametrize("parts", [1, 2, 3, 4])
def test_pairs_stay_together_in_micro_batches(parts):
    """The documented function, over what a runner's cut leaves of a batch: each part's loss is the mean over its own
    pairs, and the sum of the gradients that of the sum."""
    from pfeife_b200.utils.batch import split_args_kwargs
    model = _model()
    prefer = _documented("prefer", model=model, runner=Unscaled)
    pairs, labels, ref = _pairs(6, 12, torch.Generator().manual_seed(parts))
    each = _pair_loss(model(pairs.flatten(0, 1)).view(6, 2, 12, -1), labels, ref)
    want = [c.mean() for c in torch.tensor_split(each, parts)]
    grads = torch.autograd.grad(sum(want), list(model.parameters()))
    got = [prefer(*args) for args in split_args_kwargs((pairs, labels, ref), {}, parts)[0]]
    # rewards of some 0.1 * 66 nats, each 1e-6 of their value off, and a loss that moves no faster than they do
    assert [float(l.detach()) for l in got] == pytest.approx([float(l.detach()) for l in want], abs=2e-5)
    for p, d in zip(model.parameters(), grads):
        assert float((p.grad - d).norm()) <= 1e-4 * float(d.norm()) + 1e-9


def test_a_policy_loss_is_the_mean_of_its_micro_batch():
    from pfeife_b200.utils.batch import split_args_kwargs
    model = _model()
    reinforce = _documented("reinforce", model=model, runner=Unscaled)
    ids, labels = _batch(4, 12, torch.Generator().manual_seed(9))
    labels[2:, 6:] = -100                                  # fewer tokens in the second half
    old, adv = torch.full((4, 12), -5.5), torch.tensor([[1.0], [-1.0], [0.5], [2.0]])
    got = [reinforce(*args) for args in split_args_kwargs((ids, labels, old, adv, old), {}, 2)[0]]
    l = torch.log_softmax(model(ids).double(), -1).gather(-1, labels.clamp(min=0).unsqueeze(-1))[..., 0]
    ratio, d = (l - old).exp(), old - l
    term = -torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv) + 0.04 * (d.exp() - d - 1)
    for loss, t, n in zip(got, term.chunk(2), (labels >= 0).chunk(2)):
        assert float(loss.detach()) == pytest.approx(float((t * n).sum().detach() / n.sum()), abs=1e-5)
    assert (labels >= 0)[:2].sum() != (labels >= 0)[2:].sum()


def test_pairs_of_a_manager_whose_parts_are_in_order():
    """Sequences ordered so that each part holds its chosen ones, then their rejected ones."""
    from pfeife_b200.runtime.manager import LocalPipeManager
    torch._dynamo.reset()
    model = _model()
    option = PipeOption(device_cnt=2, batch_size=4, batch_cnt=2, cpu_test=True, no_bench_optimizer=True,
                        verbosity="warning", ctrl_timeout=60, optimizer={"type": "sgd", "lr": 0.05})
    pairs, labels, _ = _pairs(4, 16, torch.Generator().manual_seed(4))
    each = _pair_loss(model(pairs.flatten(0, 1)).view(4, 2, 16, -1), labels, torch.zeros(4, 2))
    ordered = lambda t: torch.cat([c.transpose(0, 1).flatten(0, 1) for c in t.chunk(2)])

    class Loss(LossWrapper):
        def forward(self, input, target, model=None):
            return ops.preference_loss(input, target, input.new_zeros(len(target)), beta=0.1).loss
    mgr = LocalPipeManager(model, Loss(), option)
    try:
        losses = mgr.run(ordered(labels), ordered(pairs))
        assert [float(l) for l in losses] == pytest.approx([float(c.detach().mean()) for c in each.chunk(2)], abs=2e-5)
    finally:
        mgr.close()


@pytest.mark.gpu
def test_pairs_through_a_runner():
    """The documented function as the step of a runner, two micro-batches of two pairs."""
    os.environ.setdefault("WORLD_SIZE", "1")
    os.environ.setdefault("RANK", "0")
    os.environ.setdefault("MASTER_PORT", "29879")
    from pfeife_b200 import PartialRunner, initialize_pfeife, partial_compiler
    dev = initialize_pfeife().device
    model = _model(num_layers=2).to(dev)
    ref_model = copy.deepcopy(model)
    option = PipeOption(device_cnt=1, batch_size=2, batch_cnt=2, mixed_precision="bf16", no_bench_optimizer=True,
                        verbosity="warning")
    runner = PartialRunner(option, torch.optim.SGD(model.parameters(), lr=0.0))
    torch._dynamo.reset()
    runner.set_exec_fn(_documented("prefer", model=torch.compile(model, backend=partial_compiler), runner=runner))
    pairs, labels, ref = (t.to(dev) for t in _pairs(4, 16, torch.Generator().manual_seed(7)))
    out = runner.step(pairs, labels, ref)
    torch.cuda.synchronize()
    runner.close()
    ops.unregister_params()
    with torch.no_grad():
        each = _pair_loss(ref_model(pairs.flatten(0, 1)).view(4, 2, 16, -1), labels, ref)
    # a log-probability by logits of some 1, rounded to 8 bits behind 40 roundings that add up at random: 0.03 each,
    # of 24 tokens or fewer, times beta
    for loss, want in zip(out, each.chunk(2)):
        assert float(loss.detach()) == pytest.approx(float(want.mean()), abs=0.1 * 0.03 * math.sqrt(24) * 2)
