"""Muon under data parallelism: every rank orthogonalises every matrix for itself, so ranks that
see different packs have to hold the same bits after every update."""

import multiprocessing as mp
import os
import socket

import pytest


def _free_port() -> int:
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return int(s.getsockname()[1])


def _worker(rank: int, port: int, wire: str, q) -> None:
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE="2",
                      LOCAL_RANK=str(rank), CUDA_VISIBLE_DEVICES="", OMP_NUM_THREADS="1")
    import torch

    torch.set_num_threads(1)
    from packbalance_b200.config import ModelConfig, PackBalanceConfig, TrainConfig
    from packbalance_b200.parallel.distributed import init_distributed
    from packbalance_b200.parallel.optim import FlatMuon
    from packbalance_b200.train.engine import TrainEngine

    init_distributed("cpu", timeout_s=60.0)
    torch.manual_seed(0)
    model = ModelConfig(vocab_size=101, d_model=32, n_layers=2, n_heads=4, n_kv_heads=2, d_ff=56, max_seq_len=64,
                        norm_type="layernorm")
    cfg = PackBalanceConfig(model=model, train=TrainConfig(lr=1e-2, warmup_steps=1, max_steps=6, dtype="fp32",
                                                           grad_clip=0.5, optimizer="muon", grad_reduce_dtype=wire))
    eng = TrainEngine(cfg, torch.device("cpu"))
    assert isinstance(eng.optimizer, FlatMuon)
    states = [eng.flat.data.numpy().tobytes()]
    gen = torch.Generator().manual_seed(10 + rank)
    for _ in range(4):
        ids = torch.randint(1, 101, (48,), generator=gen)
        doc = torch.tensor([0] * 20 + [1] * 28)
        labels = torch.cat([ids[1:], torch.tensor([-100])])
        labels[19] = -100
        batch = dict(input_ids=ids, labels=labels, position_ids=torch.cat([torch.arange(20), torch.arange(28)]),
                     doc_ids=doc, doc_start=torch.tensor([0] * 20 + [20] * 28))
        out = eng.step([batch], 92)
        assert bool(torch.isfinite(out["grad_norm"]))
        states.append(eng.flat.data.numpy().tobytes())
    states.append(eng.optimizer.exp_avg.numpy().tobytes())
    q.put((rank, states))


@pytest.mark.parametrize("wire", ["fp32", "bf16"])
def test_two_ranks_hold_the_same_bits(wire) -> None:
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_worker, args=(r, port, wire, q)) for r in range(2)]
    for p in procs:
        p.start()
    try:
        got = dict(q.get(timeout=180) for _ in procs)
    finally:
        for p in procs:
            p.join(timeout=30)
            if p.is_alive():
                p.kill()
    assert all(p.exitcode == 0 for p in procs)
    assert got[0] == got[1]
    assert len(set(got[0][1:5])) >= 3  # the updates did something (the first step's rate is the warm-up's)
