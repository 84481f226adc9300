"""A decoder whose embedding, feed-forward blocks and head with its loss keep less, through the runtimes: stages cut by the
planner on CPU devices, and mixed precision with registered weights, eager and under CUDA graphs, on one GPU, against
plain training of the same model and against the model of separate operators."""
import copy
import os

import pytest
import torch

from pfeife_b200 import ops
from pfeife_b200.loss import LossWrapper
from pfeife_b200.models.llama import Llama, llama_config, next_tokens
from pfeife_b200.option import PipeOption


def _model(**overrides):
    torch.manual_seed(0)
    cfg = llama_config("llama_tiny", **{"embed_scale": 2.0, "fused_mlp": True, **overrides})
    return Llama(cfg)


def _batch(n, T, g):
    ids = torch.randint(0, 256, (n, T), generator=g)
    labels = next_tokens(ids)
    labels[::2, :5] = -100
    return ids, labels


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("tied", [False, True])
def test_the_same_model_of_separate_operators(device, tied):
    model = _model(tie_embeddings=tied).to(device)
    other = Llama(llama_config("llama_tiny", tie_embeddings=tied)).to(device)
    other.load_state_dict(model.state_dict())
    ids, labels = (t.to(device) for t in _batch(3, 24, torch.Generator().manual_seed(1)))
    with torch.autocast(device, dtype=torch.bfloat16):
        loss = model(ids, labels)
        x = ops.embedding(ids, other.embed.weight) * 2.0
        cos, sin = other.rope_cos[:24], other.rope_sin[:24]
        delta = None
        for layer in other.layers:
            x, delta = layer(x, delta, cos, sin)
        y, _ = ops.rms_norm(delta, other.norm, other.cfg.rms_eps, residual=x)
        want = ops.cross_entropy(ops.linear(y, other.lm_head.weight).reshape(-1, 256), labels.reshape(-1))
    loss.backward()
    want.backward()
    # some thirty roundings to 8 bits on the way to a logit and back
    assert float(loss.detach()) == pytest.approx(float(want.detach()), rel=2e-2)
    for (name, p), q in zip(model.named_parameters(), other.parameters()):
        assert float((p.grad - q.grad).norm()) <= 30 * 2.0 ** -8 * float(q.grad.norm()), name


def test_logits_and_losses_are_of_one_model():
    model = _model()
    ids, labels = _batch(2, 16, torch.Generator().manual_seed(1))
    logits = model(ids)
    each = torch.nn.functional.cross_entropy(logits.reshape(-1, 256), labels.reshape(-1))
    assert float(model(ids, labels).detach()) == pytest.approx(float(each.detach()), abs=1e-6)
    assert next_tokens(ids)[:, :-1].equal(ids[:, 1:]) and (next_tokens(ids)[:, -1] == -100).all()


class Given(LossWrapper):
    """The model gives the loss."""

    def forward(self, input, target, model=None):
        return input


def test_stages_on_the_cpu():
    from pfeife_b200.runtime.manager import LocalPipeManager
    torch._dynamo.reset()
    model = _model()
    ref = copy.deepcopy(model)
    option = PipeOption(device_cnt=2, batch_size=4, batch_cnt=2, cpu_test=True, no_bench_optimizer=True,
                        verbosity="warning", ctrl_timeout=60, optimizer={"type": "sgd", "lr": 0.05})
    mgr = LocalPipeManager(model, Given(), option)
    ropt = torch.optim.SGD(ref.parameters(), lr=0.05)
    g = torch.Generator().manual_seed(1)
    try:
        for _ in range(2):
            ids, labels = _batch(8, 16, g)
            losses = mgr.run(labels, ids, labels)
            ropt.zero_grad()
            want = []
            for i, l in zip(ids.chunk(2), labels.chunk(2)):
                loss = ref(i, l)
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
    os.environ.setdefault("MASTER_PORT", "29881")
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

    def fn(ids, labels):
        loss = cm(ids, labels)
        runner.scaler.scale(loss).backward()
        return loss.detach()

    runner.set_exec_fn(fn)
    g = torch.Generator().manual_seed(3)
    start = [p.detach().clone() for p in ref.parameters()]
    try:
        for _ in range(4):
            ids, labels = (t.to(dev) for t in _batch(8, 16, g))
            out = runner.step(ids, labels)
            ropt.zero_grad()
            for i, (a, b) in enumerate(zip(ids.chunk(2), labels.chunk(2))):
                loss = ref(a, b)
                loss.backward()
                assert float(out[i]) == pytest.approx(float(loss.detach()), rel=1e-2)
            ropt.step()
        torch.cuda.synchronize()
        kx.check_status()
        runner.gather_params()
        graphs = len(runner.worker.graphs)
    finally:
        runner.close()
        ops.unregister_params()              # later calls of this process are of plain tensors again
    assert (graphs > 0) == cuda_graphs
    for (name, p), q, s in zip(model.named_parameters(), ref.parameters(), start):
        # the way that a weight went: some 40 roundings of 2^-9 lie between it and its gradient, four steps
        moved = (q.detach() - s).norm()
        assert float((p.detach().float() - q.detach()).norm()) <= 0.1 * float(moved) + 1e-6, name
        assert moved > 0


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_a_transformer_layer_of_images(device):
    """The feed-forward block with biases and GELU, as the UNet's transformer layers have it."""
    from pfeife_b200.models.unet import TransformerLayer
    torch.manual_seed(0)
    layer, other = (TransformerLayer(64, 4, 32, fused).to(device) for fused in (True, False))
    other.load_state_dict(layer.state_dict())
    x, ctx = torch.randn(2, 48, 64, device=device), torch.randn(2, 7, 32, device=device)
    out = []
    for m in (layer, other):
        with torch.autocast(device, dtype=torch.bfloat16):
            h, delta = m(x, None, ctx)
        y = h.float() + delta.float()
        y.square().mean().backward()
        out.append(y.detach())
    # some twenty roundings to 8 bits
    assert float((out[0] - out[1]).norm()) <= 20 * 2.0 ** -8 * float(out[1].norm())
    for (name, p), q in zip(layer.named_parameters(), other.parameters()):
        assert float((p.grad - q.grad).norm()) <= 20 * 2.0 ** -8 * float(q.grad.norm()) + 1e-6, name


@pytest.mark.timeout(900)
@pytest.mark.parametrize("mesh", [None, "-2,1"], ids=["stages", "replicas"])
def test_the_trainer_with_the_lean_operators(mesh):
    """Two ranks of the example trainer, as stages and as replicas: it runs, and the loss is a number."""
    from test_examples import COMMON, _PORT, _launch
    _PORT[0] += 40 if mesh is None else 70        # both may run at the same time
    its, loss, _ = _launch("train_llama.py", ["--model", "llama_tiny", "--block_size", "16", "--lean",
                                             "--per_device_train_batch_size", "2", "--iter_cnt", "3"] + COMMON,
                           mesh=mesh)
    assert its > 0 and loss == loss


def test_weights_that_are_read_in_16_bits_only():
    """A replica that does not own one needs no current fp32 copy of it."""
    from test_graph import capture
    model = _model(num_layers=1)
    ids, labels = _batch(2, 16, torch.Generator().manual_seed(1))
    cap, _, _ = capture(model, ids, labels)
    only = cap.shadow_only_inputs()
    assert {i.qualname for i in cap.inputs if i.is_state and i.index in only} == {
        "embed.weight", "layers.0.qkv.weight", "layers.0.o_proj.weight", "layers.0.gate_up.weight",
        "layers.0.down.weight", "lm_head.weight"}


@pytest.mark.parametrize("kind", ["embedding", "scaled_embedding"])
@pytest.mark.parametrize("precision", [torch.bfloat16, torch.float16, None], ids=str)
def test_tables_that_are_read_in_their_own_type(kind, precision):
    """The embeddings read a table's 16-bit shadow where the result has its type, else the fp32 master, which a replica
    then has to have; one such reader of several is enough."""
    from pfeife_b200.ops import functional
    from test_graph import capture
    types = [torch.bfloat16, torch.float16, torch.float32]

    class Tables(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.tables = torch.nn.ParameterList(torch.nn.Parameter(torch.randn(6, 8)) for _ in range(5))

        def forward(self, ids):
            read = getattr(ops, kind)
            out = [read(ids, t, out_dtype=d) for t, d in zip(self.tables, types)]
            out += [read(ids, self.tables[3]), read(ids, self.tables[4]), read(ids, self.tables[4], out_dtype=torch.float32)]
            return sum(y.float() for y in out)

    with functional.stage_precision(precision), torch.autocast("cpu", precision, enabled=precision is not None):
        cap, _, _ = capture(Tables(), torch.arange(4))
    only = cap.shadow_only_inputs()
    want = {types.index(precision), 3} if precision is not None else {2, 3, 4}
    assert {int(i.qualname.split(".")[-1]) for i in cap.params if i.index in only} == want


def test_weights_of_a_region_without_autocast():
    """Products that the model takes out of the stages' precision read the fp32 weights."""
    from pfeife_b200.ops import functional
    from test_graph import capture

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            for name, shape in (("before", (8, 8)), ("inside", (8, 8)), ("after", (8, 8)), ("both", (8, 8)),
                                ("gate_up", (16, 8)), ("down", (8, 8)), ("head", (6, 8))):
                setattr(self, name, torch.nn.Parameter(torch.randn(shape)))

        def forward(self, x, labels):
            x = ops.linear(ops.linear(x, self.before), self.both)
            with torch.autocast("cpu", enabled=False):
                x = ops.linear(ops.linear(x.float(), self.inside), self.both)
                x = ops.gated_mlp(x, self.gate_up, None, self.down, None)
            return ops.linear_cross_entropy(ops.linear(x, self.after), self.head, labels)

    with functional.stage_precision(torch.bfloat16), torch.autocast("cpu", torch.bfloat16):
        cap, _, _ = capture(Net(), torch.randn(3, 8), torch.arange(3))
    only = cap.shadow_only_inputs()
    assert {i.qualname for i in cap.params if i.index in only} == {"before", "after", "head"}


@pytest.mark.parametrize("own_type", [False, True], ids=["fp32 weights", "16-bit weights"])
def test_rows_of_other_replicas_come_before_a_weight_is_read(own_type, monkeypatch):
    """Row-sharded weights are completed by their first reader after an optimizer step, whether the model holds them in
    fp32 beside a 16-bit shadow or in 16 bits itself."""
    from pfeife_b200.ops import functional as Fn
    from pfeife_b200.ops import kernels as kx
    master = torch.randn(8, 4)
    lp = torch.zeros(8, 4, dtype=torch.bfloat16)
    pulled = []
    monkeypatch.setattr(kx, "gather_rows", lambda rows, *a: pulled.append(rows.copy_(master)))
    w = lp.detach() if own_type else master
    try:
        ops.register_param(master, lp, None)
        Fn.set_gather(master, Fn.GatherInfo(None, (4, 8), 2, 0, None))
        for turn in range(1, 3):
            lp.zero_()
            Fn._weight_as(w, torch.bfloat16)             # outside of a session weights are complete
            assert len(pulled) == turn - 1
            Fn.gather_session(True)
            for _ in range(2):
                assert torch.equal(Fn._weight_as(w, torch.bfloat16), master.to(torch.bfloat16)) and len(pulled) == turn
            Fn.gather_session(False)
    finally:
        Fn.gather_session(False)
        ops.unregister_params()


@pytest.mark.gpu
@pytest.mark.parametrize("own_type", [False, True], ids=["fp32 weights", "16-bit weights"])
def test_lean_operators_complete_the_weights_that_they_read(own_type, monkeypatch):
    from pfeife_b200.ops import functional as Fn
    from pfeife_b200.ops import kernels as kx
    full = [torch.randn(*s, device="cuda") * 0.2 for s in ((64, 32), (96, 32), (32, 48), (64, 32))]
    low = [t.to(torch.bfloat16) for t in full]
    held = [t.clone() for t in low]
    of = {t.data_ptr(): i for i, t in enumerate(low)}
    monkeypatch.setattr(kx, "gather_rows", lambda rows, *a: rows.copy_(held[of[rows.data_ptr()]]))
    ids, labels = (torch.randint(0, 64, (40,), device="cuda") for _ in range(2))

    def run(table, w1, w2, head):
        with torch.autocast("cuda", torch.bfloat16):
            h = ops.scaled_embedding(ids, table, 2.0, out_dtype=torch.bfloat16)
            return ops.linear_cross_entropy(ops.gated_mlp(h, w1, None, w2, None), head, labels)
    want = run(*held)
    try:
        for master, lp in zip(full, low):
            ops.register_param(master, lp, None)
            Fn.set_gather(master, Fn.GatherInfo(None, (len(lp) // 2, len(lp)), 2, 0, None))
            lp[: len(lp) // 2] = 0
        Fn.gather_session(True)
        assert torch.equal(run(*([t.detach() for t in low] if own_type else full)), want)
    finally:
        Fn.gather_session(False)
        ops.unregister_params()
