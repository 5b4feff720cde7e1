"""The native training step with layer normalisation and Muon together: model gradients against
the module path, the optimizer against its CPU form, captured steps against eager ones."""

import math
from dataclasses import replace

import pytest
import torch

from packbalance_b200.config import ModelConfig, PackBalanceConfig, TrainConfig
from packbalance_b200.data.dataset import doc_starts_from_ids
from packbalance_b200.models.llama import LlamaForCausalLM
from packbalance_b200.ops import _native
from packbalance_b200.parallel.flat import FlatParameters
from packbalance_b200.parallel.optim import FlatMuon, hidden_matrices
from packbalance_b200.train.engine import TrainEngine

pytestmark = pytest.mark.gpu
CFG = ModelConfig(vocab_size=1000, d_model=256, n_layers=2, n_heads=4, n_kv_heads=2, d_ff=512, max_seq_len=1024,
                  attention_backend="auto", ce_chunk_size=256, norm_type="layernorm")


def _batch(lengths, vocab, device="cuda", seed=0):
    gen = torch.Generator().manual_seed(seed)
    ids = torch.randint(1, vocab, (sum(lengths),), generator=gen)
    doc = torch.cat([torch.full((n,), i) for i, n in enumerate(lengths)])
    pos = torch.cat([torch.arange(n) for n in lengths])
    labels = torch.cat([ids[1:], torch.full((1,), -100)])
    labels[torch.cumsum(torch.tensor(lengths), 0) - 1] = -100
    return tuple(t.to(device) for t in (ids, labels, pos, doc))


@pytest.mark.parametrize("tied", [True, False])
@pytest.mark.parametrize("checkpointing", [False, True])
def test_native_layernorm_model_matches_module_path(tied, checkpointing):
    """Tolerances as for the RMSNorm model: bf16 activations through two layers."""
    torch.manual_seed(0)
    cfg = replace(CFG, tie_embeddings=tied)
    ids, labels, pos, doc = _batch([100, 300, 57, 555], cfg.vocab_size)
    ref = LlamaForCausalLM(replace(cfg, attention_backend="eager")).cuda()
    nat = LlamaForCausalLM(cfg).cuda()
    with torch.no_grad():
        for n, p in ref.named_parameters():
            if "norm" in n:  # weights and biases away from 1 and 0
                p.add_(0.2 * torch.randn_like(p))
            p.copy_(p.to(torch.bfloat16).float())
    nat.load_state_dict(ref.state_dict())
    nat.model.gradient_checkpointing = checkpointing
    flat = nat.flat = FlatParameters(nat)
    out_ref = ref(ids[None], labels=labels[None], position_ids=pos[None], doc_ids=doc[None])
    out_ref.loss.backward()
    flat.begin_window()
    out = nat(ids[None], labels=labels[None], position_ids=pos[None], doc_ids=doc[None])
    out.loss.backward()
    flat.finish_window()
    _native.check_status()
    n_tok = int((labels != -100).sum())
    torch.testing.assert_close(out.loss / n_tok, out_ref.loss / n_tok, atol=2e-2, rtol=1e-2)
    for (name, p_ref), p in zip(ref.named_parameters(), nat.named_parameters()):
        assert name == p[0]
        rel = (p[1].grad - p_ref.grad).norm() / (p_ref.grad.norm() + 1e-12)
        assert rel < 0.08, f"{name}: relative grad error {rel:.3f}"
    with torch.no_grad():
        logits = nat(ids[None], position_ids=pos[None], doc_ids=doc[None]).logits
        logits_ref = ref(ids[None], position_ids=pos[None], doc_ids=doc[None]).logits
    assert (logits - logits_ref).norm() / logits_ref.norm() < 0.03


def test_flat_muon_on_the_gpu_matches_the_cpu():
    """Three clipped steps.  A matrix moves by its step length times the orthogonalised
    direction, whose fp16 iteration is 3e-3 off in the Frobenius norm; the rest is fp32 AdamW.

    The two sides sum the clip norm in different orders, so their scaled gradients differ by a
    known factor 1 + d_k at step k.  An AdamW step is lr m / sqrt(v) with m = sum a_i g_i, v = sum
    c_i g_i^2 and sum a_i^2 / c_i <= 1.01 for three steps at betas 0.9 and 0.95, so |m| and sum
    |a_i g_i| are at most 1.005 sqrt(v): factors 1 + d on the g_i move m by d 1.005 sqrt(v) and
    sqrt(v) by d sqrt(v), and the step by 2.01 d lr."""
    torch.manual_seed(0)
    cfg = replace(CFG, d_ff=520)
    models = [LlamaForCausalLM(cfg) for _ in range(2)]
    models[1].load_state_dict(models[0].state_dict())
    models[0].cuda()
    flats = [FlatParameters(m) for m in models]
    lr = 1e-2
    opts = [FlatMuon(f, hidden_matrices(m), lr=lr, betas=(0.9, 0.95), weight_decay=0.1)
            for f, m in zip(flats, models)]
    gen = torch.Generator().manual_seed(1)
    apart = 0.0
    for _ in range(3):
        g = torch.randn(flats[0].numel, generator=gen) * 1e-3
        norms = []
        for f, o in zip(flats, opts):
            f.grad.copy_(g)
            norms.append(f.grad.norm())
            o.step(grad_norm=norms[-1], max_norm=0.5)
        apart = max(apart, abs(float(norms[0]) / float(norms[1]) - 1))
    _native.check_status()
    assert int(opts[0].last_skipped) == 0
    for s0, s1 in zip(flats[0].slots, flats[1].slots):
        got, want = s0.param.detach().double().cpu(), s1.param.detach().double()
        if s1 in opts[1].matrices:
            step = lr * 0.2 * math.sqrt(max(s1.shape)) * math.sqrt(min(s1.shape)) * 1.2
            assert float((got - want).norm()) <= 3 * (3e-3 * step + 2.0**-22 * float(want.norm())), s1.name
        else:
            # three AdamW steps in fp32 on both sides; sqrt and division orders differ
            tol = 3 * lr * (2.0**-20 + 2.01 * apart) + 2.0**-20 * want.abs()
            off = (got - want).abs()
            assert bool((off <= tol).all()), f"{s1.name}: {float((off / tol).max()):.3g} bounds, norms {apart:.2g} apart"
    assert torch.equal(flats[0].shadow, flats[0].data.bfloat16())
    before = flats[0].data.clone()
    opts[0].step(grad_norm=torch.tensor(math.inf, device="cuda"), max_norm=0.5)
    assert torch.equal(before, flats[0].data) and int(opts[0].last_skipped) == 1


def _engine(graphs: bool, deterministic: bool = False, **train):
    torch.manual_seed(0)
    tc = TrainConfig(lr=1e-3, warmup_steps=2, max_steps=20, grad_clip=1.0, cuda_graphs=graphs, optimizer="muon",
                     deterministic=deterministic, **train)
    return TrainEngine(PackBalanceConfig(model=CFG, train=tc), torch.device("cuda"))


def _host_batch(seed):
    ids, labels, pos, doc = _batch([200, 312, 512], CFG.vocab_size, device="cpu", seed=seed)
    return dict(input_ids=ids, labels=labels, position_ids=pos, doc_ids=doc,
                doc_start=torch.from_numpy(doc_starts_from_ids(doc.numpy())))


def test_captured_steps_match_eager_steps():
    e0, e1 = _engine(False), _engine(True)
    assert isinstance(e0.optimizer, FlatMuon) and e1.use_graphs and not e0.use_graphs
    for k in range(6):
        batch = _host_batch(k)
        for dst, src in ((e1.flat.data, e0.flat.data), (e1.flat.shadow, e0.flat.shadow),
                         (e1.optimizer.exp_avg, e0.optimizer.exp_avg),
                         (e1.optimizer.exp_avg_sq, e0.optimizer.exp_avg_sq)):
            dst.copy_(src)
        e1.flat.mark_shadow_fresh()
        before = e0.flat.data.clone()
        outs = [e.step([batch], 900) for e in (e0, e1)]
        torch.testing.assert_close(outs[1]["loss_sum"], outs[0]["loss_sum"], rtol=1e-5, atol=1e-4)
        torch.testing.assert_close(outs[1]["grad_norm"], outs[0]["grad_norm"], rtol=1e-4, atol=1e-5)
        upd = (e0.flat.data - before).norm()
        err = (e1.flat.data - e0.flat.data).norm()
        assert err <= 0.02 * upd + 1e-6, (float(err), float(upd))
    assert len(e1._graphs) == 1 and e0.optimizer.step_count == e1.optimizer.step_count == 6
    _native.check_status()


def test_deterministic_steps_repeat_bit_for_bit():
    runs = []
    for _ in range(2):
        eng = _engine(False, deterministic=True)
        try:
            for k in range(3):
                eng.step([_host_batch(k)], 900)
            runs.append(eng.flat.data.clone())
        finally:
            eng.close()
    assert torch.equal(runs[0], runs[1])
    _native.check_status()


def test_generation_with_layernorm_on_the_module_path():
    torch.manual_seed(0)
    model = LlamaForCausalLM(CFG).cuda()
    prompt = torch.randint(1, CFG.vocab_size, (2, 7), device="cuda")
    out = model.generate(prompt, max_new_tokens=5)
    cpu = LlamaForCausalLM(CFG)
    cpu.load_state_dict(model.state_dict())
    assert out.shape == (2, 12) and torch.equal(out.cpu(), cpu.generate(prompt.cpu(), max_new_tokens=5))


def test_sharding_is_refused_with_layernorm(monkeypatch):
    from packbalance_b200.train import engine

    monkeypatch.setattr(engine, "get_world_size", lambda: 2)
    monkeypatch.setattr(engine.dist, "is_initialized", lambda: True)
    cfg = PackBalanceConfig(model=CFG, train=TrainConfig(fsdp=True))
    with pytest.raises(ValueError, match="layernorm"):
        TrainEngine(cfg, torch.device("cuda"))
