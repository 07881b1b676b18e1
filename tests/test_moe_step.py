"""A training step of the mixture model with the scored router, the sorted embedding and 8-bit moments together: the layer, the model, the Trainer.

Two ways to the same layer or the same sum differ in the order of fp32 sums of at most 256 terms: 2^-14 of a tensor's 2-norm after a dozen
operations in a row; a second way in bf16 by 2^-9 for each of some ten roundings."""

import os

import pytest
import torch

from tests.dist_utils import run_distributed
from tests.test_trainer_parity import STEPS, _Interleaved, _moe_config, _weights
from torchure_b200.models.builder import build_model
from torchure_b200.objectives.autoregressive import ARObjective
from torchure_b200.ops import moe, oracle
from torchure_b200.optim.builder import build_optimizer
from torchure_b200.parallel.expert_parallel import MoELayer

ROUTER = {"score": "sigmoid", "groups": 2, "top_groups": 1, "scale": 1.5, "bias_rate": 0.01}
MODEL = dict(num_layers=2, num_heads=4, num_kv_heads=2, emb_dim=256, head_dim=64, vocab_size=512, num_experts=8, top_k=2, moe_ffn_dim=128,
             capacity_factor=0.0, experts="grouped", router=dict(ROUTER, groups=4, top_groups=2), embedding="sorted", embed_scale=16.0)


def _same(got, want, bound=2.0 ** -14):
    assert float((got.detach() - want.detach()).norm()) <= bound * float(want.detach().norm())


def test_layer_with_scores_either_way():
    """Padded buffers and grouped rows: one routing, one result, one count."""
    torch.manual_seed(0)
    old = MoELayer(16, 32, num_experts=4, top_k=2, capacity_factor=8.0, router=ROUTER)
    new = MoELayer(16, 32, num_experts=4, top_k=2, capacity_factor=0.0, experts="grouped", router=ROUTER)
    new.load_state_dict(old.state_dict())
    for layer in (old, new):
        layer.router_bias.copy_(torch.tensor([0.3, -0.3, 0.0, 0.1]))
    x = torch.randn(50, 16)
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    ya, yb = old(a), new(b)
    _same(yb, ya)
    (ya.square().sum() + old.aux_loss).backward()
    (yb.square().sum() + new.aux_loss).backward()
    _same(b.grad, a.grad)
    _same(new.router.weight.grad, old.router.weight.grad)
    assert torch.equal(old.router_counts, new.router_counts) and int(old.router_counts.sum()) == 100
    r = moe.route(old.router(x), 2, score="sigmoid", bias=old.router_bias, groups=2, top_groups=1, scale=1.5)
    assert torch.equal(r.counts, old.router_counts)
    with torch.no_grad():
        new(x)
    new.eval()
    new(x)
    assert int(new.router_counts.sum()) == 100              # only training passes count
    want = oracle.balance_bias(new.router_bias, new.router_counts, 0.01)
    new.balance()
    assert torch.equal(new.router_bias, want) and int(new.router_counts.sum()) == 0


def test_layer_refuses_what_its_router_cannot_be():
    for router in ({"score": "tanh"}, {"groups": 3}, {"bias_rate": -1.0}, {"temperature": 2.0}, {"groups": 4, "top_groups": 1}):
        with pytest.raises(ValueError):
            MoELayer(16, 32, num_experts=4, top_k=2, router=router)
    with pytest.raises(ValueError):
        build_model("qwen3_moe", dict(MODEL, embedding="hashed"))
    assert MoELayer(16, 32, num_experts=4, top_k=2, router={}).scoring is None


def test_weights_without_a_bias_load():
    plain = MoELayer(16, 32, num_experts=4, top_k=2)
    biased = MoELayer(16, 32, num_experts=4, top_k=2, router=ROUTER)
    biased.load_state_dict(plain.state_dict())
    assert "router_bias" in biased.state_dict() and (biased.router_bias == 0).all() and "router_counts" not in biased.state_dict()


def _sharded(rank, world, out):
    from torchure_b200.core.mesh import Mesh
    from torchure_b200.parallel.fsdp import FSDP

    torch.manual_seed(1)
    model = build_model("qwen3_moe", dict(MODEL, emb_dim=64, head_dim=16, moe_ffn_dim=32, router=None))
    ids = torch.arange(30).view(2, 15)
    want = model(ids).detach()
    FSDP(model, Mesh({"dp_shard": world}), "dp_shard")
    torch.save((want, model(ids).detach()), f"{out}.{rank}")


def test_lookup_of_a_sharded_table(tmp_path):
    """The table of a sharded model is gathered when its module is called: the lookup by sorting is such a call."""
    run_distributed(_sharded, 2, str(tmp_path / "out"))
    for rank in range(2):
        want, got = torch.load(tmp_path / f"out.{rank}")
        _same(got, want)


def test_a_pipeline_stage_scales_its_rows():
    class One:
        def size(self, dim):
            return 1

        def coordinate(self, dim):
            return 0

    from torchure_b200.parallel.pipeline import PipelineStage

    for kind in ("torch", "sorted"):
        torch.manual_seed(2)
        model = build_model("qwen3_moe", dict(MODEL, embedding=kind))
        assert model.lm_head.weight is model.token_emb.weight and "token_emb.weight" in model.state_dict()
        ids = torch.arange(12).view(1, 12)
        with torch.no_grad():
            _same(PipelineStage(model, One())(ids), model(ids))


def _run(rank, world, cfg, home, out, emulate_world):
    os.environ["TORCHURE_B200_HOME"] = home
    from torchure_b200.train.trainer import Trainer

    tr = Trainer(cfg, rank, rank, world, benchmark=True, device="cpu")
    if emulate_world:
        tr.prefetcher = _Interleaved(cfg, emulate_world)
    hist = tr.train_n_step_test(STEPS)
    buffers = {n: b.clone() for n, b in tr.model.named_buffers() if "router" in n}
    torch.save({"hist": hist, "params": _weights(tr), "buffers": buffers}, f"{out}.{rank}")


def _config(world, accumulation, bits=32, **kw):
    cfg = _moe_config(world, accumulation, **kw)
    cfg["model"]["config"].update(experts="grouped", router=ROUTER, embedding="sorted", embed_scale=2.0)
    cfg["optimizer"]["config"].update(state_bits=bits)
    return cfg


def test_spread_over_ranks_the_bias_is_that_of_one_process(tmp_path):
    run_distributed(_run, 1, _config(1, 2), str(tmp_path), str(tmp_path / "one.pt"), 2, timeout_s=240)
    run_distributed(_run, 2, _config(2, 1, mesh={"dp": 1, "ep": 2}), str(tmp_path), str(tmp_path / "ep.pt"), 0, timeout_s=240)
    one = torch.load(f"{tmp_path}/one.pt.0")
    parts = [torch.load(f"{tmp_path}/ep.pt.{r}") for r in range(2)]
    for x, y in zip(parts[0]["hist"], one["hist"]):
        assert abs(x["loss"] - y["loss"]) < 1e-4 * max(1.0, abs(y["loss"])), (x, y)
    assert sum(float(b.abs().sum()) for n, b in one["buffers"].items() if n.endswith("router_bias")) > 0
    for name, b in one["buffers"].items():
        assert torch.equal(parts[0]["buffers"][name], parts[1]["buffers"][name]), name
        if name.endswith("router_bias"):
            # a step's move may differ where a token's choice went the other way in a tie of fp32 sums: a few, never most
            assert ((parts[0]["buffers"][name] - b).abs() < 1e-6).float().mean() >= 0.75


def test_replicas_with_8_bit_moments_stay_equal(tmp_path):
    run_distributed(_run, 2, _config(2, 1, bits=8), str(tmp_path), str(tmp_path / "dp.pt"), 0, timeout_s=240)
    a, b = (torch.load(f"{tmp_path}/dp.pt.{r}") for r in range(2))
    for kind in ("params", "buffers"):
        assert all(torch.equal(a[kind][n], b[kind][n]) for n in a[kind])


def _resume(rank, world, home, out):
    os.environ["TORCHURE_B200_HOME"] = home
    from torchure_b200.train.trainer import Trainer

    straight = Trainer(_config(1, 2, 8, run_name="straight"), rank, rank, world, device="cpu")
    straight.train()
    first = Trainer(_config(1, 2, 8, run_name="resumed", save_steps=3), rank, rank, world, device="cpu")
    first.num_train_steps = 3
    first.train()
    second = Trainer(_config(1, 2, 8, run_name="resumed", resume="auto"), rank, rank, world, device="cpu")
    assert second.start_step == 3
    second.train()
    states = [[{n: v for n, v in st.items()} for st in tr.optimizer.state.values()] for tr in (straight, second)]
    torch.save({"a": straight.model.state_dict(), "b": second.model.state_dict(), "states": states}, out)


def test_resume_with_8_bit_moments_and_a_bias_is_exact(tmp_path):
    run_distributed(_resume, 1, str(tmp_path), str(tmp_path / "r.pt"), timeout_s=240)
    got = torch.load(tmp_path / "r.pt")
    assert any(n.endswith("router_bias") and v.abs().sum() > 0 for n, v in got["a"].items())
    assert all(torch.equal(got["a"][n], got["b"][n]) for n in got["a"])
    for x, y in zip(*got["states"]):
        assert set(x) == set(y) and x["exp_avg"].dtype == torch.uint8 and all(torch.equal(x[n], y[n]) for n in x)


@pytest.mark.gpu
def test_layer_on_the_gpu_against_the_plain_one():
    for bits in (16, 8):
        torch.manual_seed(1)
        layer = MoELayer(256, 192, num_experts=8, top_k=2, capacity_factor=0.0, experts="grouped", act_bits=bits, router=dict(ROUTER, groups=4, top_groups=2)).cuda()
        layer.router_bias.copy_(torch.randn(8) * 0.1)
        plain = MoELayer(256, 192, num_experts=8, top_k=2, capacity_factor=0.0, experts="grouped", router=dict(ROUTER, groups=4, top_groups=2))
        plain.load_state_dict(layer.state_dict())
        x = torch.randn(300, 256).bfloat16().float()
        a, b = x.cuda().requires_grad_(), x.clone().requires_grad_()
        out, want = layer(a), plain(b)
        (out.square().sum() + layer.aux_loss).backward()
        (want.square().sum() + plain.aux_loss).backward()
        # the GPU's rows, weights and products are bf16, some ten roundings in a row; in 8 bits gate and up 0.04 more.  Logits are fp32 on
        # both sides: a token whose choice is a tie of their sums could go either way, and none of 300 does
        assert torch.equal(layer.router_counts.cpu(), plain.router_counts)
        slack = 0.04 if bits == 8 else 0.0
        _same(out.cpu(), want, 10 * 2.0 ** -9)
        for name in ("w_gate", "w_up", "w_down"):
            _same(getattr(layer, name).grad.cpu(), getattr(plain, name).grad, 10 * 2.0 ** -9 + slack)
        _same(a.grad.cpu(), b.grad, 10 * 2.0 ** -9 + slack)


@pytest.mark.gpu
def test_a_training_step_of_everything():
    """Lookup, routers, grouped experts, loss head, 8-bit step and bias, as the Trainer calls them one after the other; a second model that runs the
    embedding in PyTorch and keeps 32-bit moments sees the same first loss and nearly the same gradients."""
    model = build_model("qwen3_moe", MODEL).cuda()
    model.init_weights()
    other = build_model("qwen3_moe", dict(MODEL, embedding="torch")).cuda()
    other.load_state_dict(model.state_dict())
    opt = build_optimizer(model, "adamw", dict(lr=1e-3, weight_decay=0.1, betas=[0.9, 0.95], fused=True, state_bits=8))
    ids = torch.randint(0, 512, (2, 128), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    objective = ARObjective(fused_linear_ce=True, ce_chunk_size=256)
    losses = []
    for m in (model, other):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            losses.append(objective.compute_loss(m, {"input_ids": ids, "labels": ids}))
        losses[-1].backward()
    assert torch.equal(losses[0], losses[1])          # the lookups' rows have the same bits
    for (name, p), q in zip(model.named_parameters(), other.parameters()):
        _same(p.grad, q.grad, 10 * 2.0 ** -9)
    for _ in range(3):
        opt.step()
        opt.zero_grad()
        model.balance_routers()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = objective.compute_loss(model, {"input_ids": ids, "labels": ids})
        loss.backward()
        assert torch.isfinite(loss) and all(torch.isfinite(p.grad).all() for p in model.parameters())
    assert all(st["exp_avg"].dtype == torch.uint8 for st in opt.state.values())
    assert all(float(b.ffn.router_bias.abs().max()) > 0 for b in model.blocks)


@pytest.mark.gpu
def test_trainer_runs_the_shipped_configuration(tmp_path, monkeypatch):
    """The shipped config with its model made small: steps, a checkpoint, and a second run that goes on from it."""
    import json

    monkeypatch.setenv("TORCHURE_B200_HOME", str(tmp_path))
    monkeypatch.setenv("MASTER_ADDR", "127.0.0.1")
    from tests.dist_utils import free_port
    from torchure_b200.train.trainer import Trainer

    monkeypatch.setenv("MASTER_PORT", str(free_port()))
    with open(os.path.join(os.path.dirname(__file__), "..", "configs", "qwen3_moe_64x_synthetic_dp1.json")) as f:
        cfg = json.load(f)
    cfg["model"]["config"].update(num_layers=2, num_heads=4, num_kv_heads=2, emb_dim=256, vocab_size=2048, moe_ffn_dim=64)
    cfg["data"].update(seq_len=256, eos_id=0)
    cfg["checkpointing"]["save_steps"] = 2
    cfg["optimizer"]["scheduler"]["total_steps"] = 4
    import torch.distributed as dist

    if not dist.is_initialized():
        dist.init_process_group("nccl", rank=0, world_size=1)
    try:
        tr = Trainer(cfg, 0, 0, 1)
        tr.num_train_steps = 2
        tr.train()
        tr.check_device_errors()
        bias = tr.model.blocks[0].ffn.router_bias.clone()
        assert float(bias.abs().max()) > 0 and all(st["exp_avg"].dtype == torch.uint8 for st in tr.optimizer.state.values())
        cfg["checkpointing"]["resume"] = "auto"
        again = Trainer(cfg, 0, 0, 1)
        assert again.start_step == 2 and torch.equal(again.model.blocks[0].ffn.router_bias, bias)
        for p, q in zip(tr.optimizer.state.values(), again.optimizer.state.values()):
            assert all(torch.equal(p[n], q[n]) for n in p)
        history = again.train_n_step_test(2)
        assert all(h["loss"] == h["loss"] for h in history)
    finally:
        dist.destroy_process_group()


@pytest.mark.gpu
def test_dense_trainer_with_8_bit_moments_in_a_graph(tmp_path, monkeypatch):
    """The dense model on the kernel engine, its step captured: the shadow weights follow the masters, the replayed step counts its steps, and a run
    without the graph ends nearly where this one does (the engine's gradients differ in the order of their sums, and an update is at most
    some lr a step)."""
    monkeypatch.setenv("TORCHURE_B200_HOME", str(tmp_path))
    monkeypatch.setenv("MASTER_ADDR", "127.0.0.1")
    import torch.distributed as dist

    from tests.dist_utils import free_port
    from tests.tiny import parity_config
    from torchure_b200.train.trainer import Trainer

    monkeypatch.setenv("MASTER_PORT", str(free_port()))
    if not dist.is_initialized():
        dist.init_process_group("nccl", rank=0, world_size=1)
    try:
        ends = []
        for graph in (False, True):
            cfg = parity_config(world=1, steps=8, accumulation=1)
            cfg["model"]["config"].update(num_layers=2, num_heads=4, num_kv_heads=2, emb_dim=256, head_dim=128, vocab_size=1024, ffn_dim=512)
            cfg["optimizer"]["config"].update(fused=True, state_bits=8)
            cfg.update(cuda_graph=graph, cuda_graph_warmup=2)
            tr = Trainer(cfg, 0, 0, 1, benchmark=True)
            history = tr.train_n_step_test(6)
            tr.check_device_errors()
            assert all(h["loss"] == h["loss"] for h in history) and (tr._graph is not None) == graph
            states = tr.optimizer.state
            assert all(st["exp_avg"].dtype == torch.uint8 and float(st["step"]) == 6 for st in states.values())
            for p, shadow in tr.model.engine().shadow_pairs():
                assert torch.equal(shadow.reshape(p.shape), p.detach().bfloat16())
            ends.append([p.detach().clone() for p in tr.model.parameters()])
        for a, b in zip(*ends):
            assert float((a - b).abs().max()) <= 6 * 2 * 3e-4
    finally:
        dist.destroy_process_group()


def test_layer_whose_groups_count_by_their_largest_score():
    torch.manual_seed(3)
    router = dict(score="softmax", groups=4, top_groups=2, group_scores=1, normalize=False, scale=4.0)
    layers = [MoELayer(16, 32, num_experts=8, top_k=2, capacity_factor=8.0, router=router),
              MoELayer(16, 32, num_experts=8, top_k=2, capacity_factor=0.0, experts="grouped", router=router)]
    layers[1].load_state_dict(layers[0].state_dict())
    x = torch.randn(60, 16)
    _same(layers[1](x), layers[0](x))
    logits = layers[0].router(x).detach()
    mine = moe.route(logits, 2, **router)
    assert not torch.equal(mine.counts, moe.route(logits, 2, **dict(router, group_scores=2)).counts)
    with pytest.raises(ValueError):
        MoELayer(16, 32, num_experts=8, top_k=2, router=dict(router, group_scores=3))


@pytest.mark.gpu
def test_replayed_steps_of_the_dense_trainer_move_as_eager_ones(tmp_path, monkeypatch):
    """The dense model on the kernel engine with 8-bit moments, its step captured, against a run without the graph, measured by the way that the weights
    go.  Gradients of the two runs differ in the order of fp32 sums, some 2^-20 of a tensor's norm, so that an element's update, m over the root of
    v, is another only where its gradient is that small beside the rest, or where a code falls to the other side, by an eighth, for as rare an
    element: far less than a sixteenth of the way.  A step that a replay leaves out, or takes twice, is a sixth of it."""
    monkeypatch.setenv("TORCHURE_B200_HOME", str(tmp_path))
    monkeypatch.setenv("MASTER_ADDR", "127.0.0.1")
    import torch.distributed as dist

    from tests.dist_utils import free_port
    from tests.tiny import parity_config
    from torchure_b200.train.trainer import Trainer

    monkeypatch.setenv("MASTER_PORT", str(free_port()))
    if not dist.is_initialized():
        dist.init_process_group("nccl", rank=0, world_size=1)
    try:
        runs = []
        for graph in (False, True):
            cfg = parity_config(world=1, steps=8, accumulation=1)
            cfg["model"]["config"].update(num_layers=2, num_heads=4, num_kv_heads=2, emb_dim=256, head_dim=128, vocab_size=1024, ffn_dim=512)
            cfg["optimizer"]["config"].update(fused=True, state_bits=8)
            cfg.update(cuda_graph=graph, cuda_graph_warmup=2)
            tr = Trainer(cfg, 0, 0, 1, benchmark=True)
            places = [[p.detach().clone() for p in tr.model.parameters()]]
            losses = []
            for _ in range(6):
                losses += [h["loss"] for h in tr.train_n_step_test(1)]
                places.append([p.detach().clone() for p in tr.model.parameters()])
            tr.check_device_errors()
            assert (tr._graph is not None) == graph
            runs.append((places, losses))
        (eager, le), (replayed, lr) = runs
        assert all(torch.equal(p, q) for p, q in zip(eager[0], replayed[0]))
        for t in range(1, 7):
            for start, was, is_, other in zip(eager[0], replayed[t - 1], replayed[t], eager[t]):
                assert not torch.equal(was, is_), t
                assert float((is_ - other).norm()) <= float((other - start).norm()) / 16, t
        # losses of weights that are as near, in bf16 products: a few units of 2^-9 of a logit of order one
        assert all(abs(x - y) <= 2.0 ** -8 for x, y in zip(le, lr)), (le, lr)
    finally:
        dist.destroy_process_group()
