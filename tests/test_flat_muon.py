"""FlatMuon and the layer-norm decoder on the CPU: update, state, checkpoints, configuration."""

import math
from dataclasses import replace
from pathlib import Path

import pytest
import torch

from packbalance_b200.config import ModelConfig, PackBalanceConfig, TrainConfig, apply_overrides
from packbalance_b200.data.dataset import PackedDataset
from packbalance_b200.data.packer import build_packs
from packbalance_b200.models.llama import LayerNorm, LlamaForCausalLM, RMSNorm
from packbalance_b200.ops.reference import newton_schulz_reference
from packbalance_b200.parallel.flat import FlatParameters
from packbalance_b200.parallel.optim import FlatAdamW, FlatMuon, hidden_matrices
from packbalance_b200.train.checkpoint import load_checkpoint, save_checkpoint
from packbalance_b200.train.engine import TrainEngine


def _make(cfg, seed=0, **kw):
    torch.manual_seed(seed)
    model = LlamaForCausalLM(cfg)
    flat = FlatParameters(model)
    return model, flat, FlatMuon(flat, hidden_matrices(model), lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1, **kw)


def test_hidden_matrices_are_the_projections(model_cfg: ModelConfig) -> None:
    model, flat, opt = _make(replace(model_cfg, norm_type="layernorm"))
    names = {s.name for s in opt.matrices}
    assert len(names) == 7 * model_cfg.n_layers and all("proj" in n for n in names)
    assert {s.name for s in opt.others} == {n for n, _ in model.named_parameters()} - names
    assert opt.exp_avg_sq.numel() == sum(s.numel for s in opt.others)


@pytest.mark.parametrize("clip", [0.0, 0.5])
def test_matrices_take_muon_and_the_rest_adamw(model_cfg: ModelConfig, clip) -> None:
    model, flat, opt = _make(model_cfg)
    model2 = LlamaForCausalLM(model_cfg)
    model2.load_state_dict(model.state_dict())
    flat2 = FlatParameters(model2)
    adam = FlatAdamW(flat2, lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1)
    gen = torch.Generator().manual_seed(3)
    mom = {s.name: torch.zeros(s.shape) for s in opt.matrices}
    want = {s.name: s.param.detach().clone() for s in opt.matrices}
    for _ in range(3):
        g = torch.randn(flat.numel, generator=gen) * 1e-2
        flat.grad.copy_(g)
        flat2.grad.copy_(g)
        norm = flat.grad.norm() if clip else None
        scale = min(1.0, clip / (float(norm) + 1e-6)) if clip else 1.0
        opt.step(grad_norm=norm, max_norm=clip)
        adam.step(grad_norm=norm, max_norm=clip)
        for s in opt.matrices:
            gk = s.param.grad * scale
            mom[s.name] += 0.05 * (gk - mom[s.name])
            u = gk + 0.95 * (mom[s.name] - gk)
            o = newton_schulz_reference(u.double(), 5, (3.4445, -4.7750, 2.0315), 1e-7).float()
            want[s.name] = want[s.name] * (1 - 1e-2 * 0.1) - 1e-2 * 0.2 * math.sqrt(max(s.shape)) * o
    for s in opt.matrices:
        torch.testing.assert_close(s.param.detach(), want[s.name], atol=2e-5, rtol=1e-4)
    for s, s2 in zip(flat.slots, flat2.slots):
        if s in opt.others:
            torch.testing.assert_close(s.param, s2.param, atol=1e-7, rtol=1e-6)


def test_nonfinite_norm_skips_update(model_cfg: ModelConfig) -> None:
    _, flat, opt = _make(model_cfg)
    before = flat.data.clone()
    flat.grad.fill_(1.0)
    opt.step(grad_norm=torch.tensor(math.nan), max_norm=1.0)
    assert torch.equal(before, flat.data) and int(opt.last_skipped) == 1 and opt.step_count == 0
    opt.step(grad_norm=torch.tensor(1.0), max_norm=1.0)
    assert not torch.equal(before, flat.data) and int(opt.last_skipped) == 0


def test_a_step_without_a_norm_clears_the_skip(model_cfg: ModelConfig) -> None:
    _, flat, opt = _make(model_cfg)
    flat.grad.fill_(1.0)
    opt.step(grad_norm=torch.tensor(math.inf), max_norm=1.0)
    assert int(opt.last_skipped) == 1
    opt.step()
    assert int(opt.last_skipped) == 0 and opt.step_count == 1


def test_checkpoint_round_trip_continues_the_run(tmp_path: Path, model_cfg: ModelConfig) -> None:
    model, flat, opt = _make(model_cfg)
    gen = torch.Generator().manual_seed(4)
    grads = [torch.randn(flat.numel, generator=gen) for _ in range(3)]
    for g in grads[:2]:
        flat.grad.copy_(g)
        opt.step()
    d = save_checkpoint(model, opt, 2, tmp_path, fsdp=False)
    model2, flat2, opt2 = _make(model_cfg, seed=9)
    assert load_checkpoint(d, model2, opt2, fsdp=False, device=torch.device("cpu"))["step"] == 2
    assert opt2.step_count == 2
    for f, o in ((flat, opt), (flat2, opt2)):
        f.grad.copy_(grads[2])
        o.step()
    assert torch.equal(flat.data, flat2.data)


def test_refuses_state_of_another_optimizer_and_bad_matrices(model_cfg: ModelConfig) -> None:
    model, flat, opt = _make(model_cfg)
    adam = FlatAdamW(FlatParameters(LlamaForCausalLM(model_cfg)))
    before = opt.exp_avg.clone()
    with pytest.raises(ValueError, match="another optimizer"):
        opt.load_state_dict(adam.state_dict())
    assert torch.equal(opt.exp_avg, before)
    with pytest.raises(ValueError, match="not a matrix"):
        FlatMuon(flat, [model.model.norm.weight])
    with pytest.raises(ValueError, match="not parameters"):
        FlatMuon(flat, [torch.nn.Parameter(torch.ones(2, 2))])


def test_adamw_refuses_the_state_of_muon_before_anything_changes(model_cfg: ModelConfig) -> None:
    _, flat, muon = _make(model_cfg)
    flat.grad.fill_(1e-3)
    muon.step()
    adam = FlatAdamW(FlatParameters(LlamaForCausalLM(model_cfg)), lr=0.5)
    kept = [t.clone() for t in (adam.exp_avg, adam.exp_avg_sq)], dict(adam.param_groups[0])
    with pytest.raises(ValueError, match="another optimizer"):
        adam.load_state_dict(muon.state_dict())
    for got, want in zip((adam.exp_avg, adam.exp_avg_sq), kept[0]):
        assert torch.equal(got, want)
    assert {k: v for k, v in adam.param_groups[0].items() if k != "params"} == \
        {k: v for k, v in kept[1].items() if k != "params"}
    assert adam.step_count == 0


def test_norm_type_builds_layer_norms(model_cfg: ModelConfig) -> None:
    model = LlamaForCausalLM(replace(model_cfg, norm_type="layernorm"))
    norms = [m for m in model.modules() if isinstance(m, LayerNorm)]
    assert len(norms) == 2 * model_cfg.n_layers + 1 and not any(isinstance(m, RMSNorm) for m in model.modules())
    assert not any(isinstance(m, LayerNorm) for m in LlamaForCausalLM(model_cfg).modules())
    x = torch.randn(3, model_cfg.d_model)
    want = torch.nn.functional.layer_norm(x, (model_cfg.d_model,), eps=model_cfg.norm_eps)
    torch.testing.assert_close(norms[0](x), want, atol=1e-5, rtol=1e-5)


@pytest.mark.parametrize("override,message", [
    ("model.norm_type=batchnorm", "norm_type"),
    ("train.optimizer=sgd", "optimizer"),
    ("train.muon_momentum=1.0", "muon_momentum"),
    ("train.muon_steps=0", "muon_steps"),
])
def test_configuration_refusals(override, message) -> None:
    with pytest.raises(ValueError, match=message):
        apply_overrides(PackBalanceConfig(), [override])


def test_muon_with_sharding_is_refused(model_cfg: ModelConfig) -> None:
    with pytest.raises(ValueError, match="not with fsdp"):
        TrainConfig(optimizer="muon", fsdp=True)
    cfg = PackBalanceConfig(model=model_cfg, train=TrainConfig(optimizer="muon"))
    cfg.train.fsdp = True  # as the command line sets it
    with pytest.raises(ValueError, match="muon"):
        TrainEngine(cfg, torch.device("cpu"))


def test_engine_steps_with_both_options(store, data_cfg, model_cfg, flop_model) -> None:
    packs = build_packs(store, data_cfg, flop_model)[:2]
    ds = PackedDataset(store, packs, data_cfg)
    batches = [ds[i] for i in range(2)]
    tokens = sum(p.tokens for p in packs)
    cfg = PackBalanceConfig(model=replace(model_cfg, norm_type="layernorm"), data=data_cfg,
                            train=TrainConfig(lr=1e-2, warmup_steps=1, max_steps=5, dtype="fp32", optimizer="muon"))
    torch.manual_seed(0)
    eng = TrainEngine(cfg, torch.device("cpu"))
    assert isinstance(eng.optimizer, FlatMuon)
    before = {n: p.detach().clone() for n, p in eng.model.named_parameters()}
    for _ in range(2):  # the first step's learning rate is the warm-up's 0
        out = eng.step(batches, tokens)
        assert bool(torch.isfinite(out["grad_norm"]))
    for n, p in eng.model.named_parameters():
        assert not torch.equal(p, before[n]), n
