"""Per-token losses of a language model under data parallelism: two gloo ranks on the CPU.

Ranks have batches of their own; after one backward pass both must hold the
mean of their gradients, whichever wrapper and entry point was used, and a
differentiable call past the wrapper is refused.
"""

from __future__ import annotations

import datetime
import os
import socket

import pytest
import torch

from koochak_b200.models import GPT2, Llama


def _port() -> int:
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _model(kind):
    torch.manual_seed(3)
    if kind == "gpt2":
        return GPT2(n_layer=1, n_head=1, n_embd=64, vocab_size=97, block_size=16)
    return Llama(n_layer=1, n_head=1, dim=64, ffn_dim=48, vocab_size=97, max_seq_len=16)


def _batch(rank):
    gen = torch.Generator().manual_seed(rank + 20)
    idx = torch.randint(0, 97, (2, 12), generator=gen)
    ids = torch.randint(0, 97, (2, 12, 4), generator=gen)
    return idx, torch.randint(0, 97, (2, 12), generator=gen), ids, torch.randn(2, 12, 4, generator=gen)


def _loss(model, rank, method):
    """A distillation step with a policy term: two forward passes before one backward pass."""

    idx, tokens, ids, t = _batch(rank)
    if method:
        kd = model(idx, method="distillation_loss", teacher_ids=ids, teacher_logits=t, temperature=2.0)
        lp = model(idx, method="token_logprobs", tokens=tokens, ignore_index=int(tokens[0, 0]))
    else:
        kd = model.distillation_loss(idx, ids, t, temperature=2.0)
        lp = model.token_logprobs(idx, tokens, ignore_index=int(tokens[0, 0]))
    return kd - 0.1 * lp.logprobs.mean() - 0.01 * lp.entropy.mean()


def _grads(model):
    return {n.removeprefix("module."): p.grad.clone() for n, p in model.named_parameters()}


def _step_fn(model, batch, ctx):
    return {"loss": model(batch["idx"], method="distillation_loss", teacher_ids=batch["ids"], teacher_logits=batch["t"])}


class _Rows(torch.utils.data.IterableDataset):
    def __init__(self, rank):
        self.rank = rank

    def __iter__(self):
        while True:
            idx, _, ids, t = _batch(self.rank)
            yield {"idx": idx, "ids": ids, "t": t}


def _worker(rank, world, port, out, kind):
    import torch.distributed as dist
    from torch.nn.parallel import DistributedDataParallel

    from koochak_b200.loop import training_loop
    from koochak_b200.optim.build import build_optimizer
    from koochak_b200.parallel.ddp import DataParallel

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world))
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=60))
    try:
        got = {}
        for name, wrap, method in (("methods", DataParallel, False), ("forward", DataParallel, True),
                                   ("torch", DistributedDataParallel, True)):
            model = wrap(_model(kind))
            _loss(model, rank, method).backward()
            got[name] = _grads(model)
        dp = DataParallel(_model(kind))
        idx, tokens, ids, t = _batch(rank)
        for call in (lambda: dp.module.distillation_loss(idx, ids, t), lambda: dp.module.token_logprobs(idx, tokens),
                     lambda: dp.module.logits(idx)):
            with pytest.raises(RuntimeError, match="past its DataParallel wrapper"):
                call()
        with torch.no_grad():
            torch.testing.assert_close(dp.module.logits(idx), dp.logits(idx), rtol=0, atol=0)
        with dp.no_sync():
            _loss(dp.module, rank, False).backward()
        got["local"] = _grads(dp)

        seen = []

        def step_fn(model, batch, ctx):
            seen.append(type(model).__name__)
            if model.require_backward_grad_sync:  # the last micro-step of an update
                with pytest.raises(RuntimeError, match="past its DistributedDataParallel wrapper"):
                    model.module.logits(batch["idx"])
            return _step_fn(model, batch, ctx)

        model = _model(kind)
        cfg = {"max_steps": 3, "grad_accum": 2, "log_every": 1000, "eval_every": 0, "ckpt_every": 3, "amp": "fp32",
               "grad_clip_norm": 1.0, "out_dir": os.path.join(out, "ckpt"), "keep_last_k": 1, "ddp": True,
               "seed": 5, "warn_unsharded": False}
        training_loop(model=model, dataset=_Rows(rank), step_fn=step_fn,
                      optimizer=build_optimizer(model, {"name": "adamw", "lr": 1e-3}), train_cfg=cfg, resume="none")
        assert seen == ["DistributedDataParallel"] * 6
        got["trained"] = {k: v.detach().clone() for k, v in model.state_dict().items()}
        torch.save(got, os.path.join(out, f"rank{rank}.pt"))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("kind", ["gpt2", "llama"])
def test_two_ranks_hold_the_mean_gradient(tmp_path, kind):
    import torch.multiprocessing as mp

    mp.spawn(_worker, args=(2, _port(), str(tmp_path), kind), nprocs=2, join=True)
    a, b = (torch.load(tmp_path / f"rank{r}.pt") for r in range(2))
    for name in ("methods", "forward", "torch"):
        for n in a["local"]:
            assert torch.equal(a[name][n], b[name][n]), (name, n)
            # (x + y) / 2 in fp32 in either form: a rounding of the sum, and of each half
            mean = (a["local"][n] + b["local"][n]) / 2
            size = a["local"][n].abs() + b["local"][n].abs()
            assert ((a[name][n] - mean).abs() <= size * 2.0**-22 + 1e-30).all(), (name, n)
    assert any(not torch.equal(a["local"][n], b["local"][n]) for n in a["local"])
    start = _model(kind).state_dict()
    for k, v in a["trained"].items():
        assert torch.equal(v, b["trained"][k])
    assert any(not torch.equal(v, start[k]) for k, v in a["trained"].items())


@pytest.mark.parametrize("kind", ["gpt2", "llama"])
def test_calls_by_way_of_forward(kind):
    """The same results as the methods, and refusals of calls that mean nothing."""

    model = _model(kind)
    idx, tokens, ids, t = _batch(0)
    assert torch.equal(_loss(model, 0, True), _loss(model, 0, False))
    assert torch.equal(model(idx, method="logits"), model.logits(idx))
    for bad, error in ((dict(method="generate"), ValueError), (dict(method="logits", targets=tokens), ValueError),
                       (dict(tokens=tokens), TypeError), (dict(method="logits", tokens=tokens), TypeError)):
        with pytest.raises(error):
            model(idx, **bad)
    assert model(idx, tokens).ndim == 0 and model(idx).shape == (2, 12, 97)


def test_a_wrapper_of_another_model_has_no_losses(monkeypatch):
    import torch.distributed as dist

    from koochak_b200.parallel.ddp import DataParallel

    monkeypatch.setenv("MASTER_ADDR", "127.0.0.1")
    monkeypatch.setenv("MASTER_PORT", str(_port()))
    dist.init_process_group("gloo", rank=0, world_size=1)
    try:
        dp = DataParallel(torch.nn.Linear(3, 3))
        with pytest.raises(AttributeError, match="Linear has no logits"):
            dp.logits(torch.zeros(1, 3))
    finally:
        dist.destroy_process_group()
