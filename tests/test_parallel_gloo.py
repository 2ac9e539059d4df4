"""Data-parallel semantics on CPU with two gloo ranks: the collectives of parallel.py composed with
the oracle's compute must reproduce the single-process result on the concatenated batch (QAT scales
via MAX, clamped spectral terms via global sums, gradients via SUM)."""
import os
import sys

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _worker(rank, world, port, ret):
    sys.path.insert(0, ROOT)
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        import importlib.util
        spec = importlib.util.spec_from_file_location("dpd_parallel", os.path.join(ROOT, "6g-pa-gan-dpd_amd", "parallel.py"))
        par = importlib.util.module_from_spec(spec); spec.loader.exec_module(par)
        from oracle import generator as og, spectral as osp
        dp = par.DataParallel()
        assert dp.enabled and dp.world == world and dp.rank == rank
        torch.manual_seed(0)
        B, S = 6, 69
        iq = torch.randn(B, S, 2) * 0.3
        tgt = torch.randn(B, S - 5, 2) * 0.3
        params = {k: torch.randn(s) * 0.2 for k, s in zip(og.PARAM_KEYS, [(32, 30), (32,), (16, 32), (16,), (2, 16), (2,)])}
        lo, hi = dp.shard_rows(B)
        assert (lo, hi) == ((0, 3) if rank == 0 else (3, 6))

        # --- QAT scales: per-stage abs-max with MAX across ranks == abs-max of the whole batch
        f_loc = og.tap_assembly(iq[lo:hi]).reshape(-1, 30)
        m = dp.max_(f_loc.abs().max().reshape(1).clone())
        assert torch.equal(m[0], og.tap_assembly(iq).abs().max())

        # --- loss with clamped batch means from global sums; gradients summed over ranks
        pp = {k: v.clone().requires_grad_(True) for k, v in params.items()}
        out = og.gen_forward(iq[lo:hi], pp)
        t = tgt[lo:hi]
        l1 = (out - t).abs().mean()
        evm_db = osp.evm(out, t)
        lo_db, up_db = osp.acpr(out)
        sums = dp.global_sum(torch.stack([l1 / world, evm_db.sum() / B, lo_db.sum() / B, up_db.sum() / B]))
        loss = 50 * sums[0] + 20 * torch.clamp((sums[1] + 40) / 40, 0, 2) + 10 * torch.clamp((torch.max(sums[2], sums[3]) + 50) / 50, 0, 2)
        loss.backward()
        plist = [pp[k] for k in og.PARAM_KEYS]
        dp.sum_grads_(plist)

        pr = {k: v.clone().requires_grad_(True) for k, v in params.items()}
        ref_total, _ = osp.spectral_loss(og.gen_forward(iq, pr), tgt)
        ref_total.backward()
        assert torch.allclose(loss.detach(), ref_total.detach(), rtol=1e-5)
        for k in og.PARAM_KEYS:
            assert torch.allclose(pp[k].grad, pr[k].grad, rtol=2e-4, atol=1e-6), k
        # mean_ / sum_
        v = torch.tensor([float(rank + 1)])
        assert dp.mean_(v.clone()).item() == 1.5 and dp.sum_(v.clone()).item() == 3.0
        # --- an odd number of rows: every rank must get the same number of rows, batch size and steps (each step
        # issues collectives; a rank with one step more would wait in them for ever)
        spec = importlib.util.spec_from_file_location("dpd_train", os.path.join(ROOT, "6g-pa-gan-dpd_amd", "train.py"))
        trn = importlib.util.module_from_spec(spec); spec.loader.exec_module(trn)
        rows = torch.arange(1023 * 2, dtype=torch.float32).reshape(1023, 1, 2)
        x_loc, t_loc, batch = trn.shard_equal(rows, rows, 256, dp.world, dp.rank)
        steps = len(range(0, x_loc.shape[0] - batch + 1, batch))
        shape = torch.tensor([x_loc.shape[0], batch, steps], dtype=torch.float32)
        assert torch.equal(dp.max_(shape.clone()), shape) and torch.equal(-dp.max_(-shape.clone()), shape)
        assert steps == 1 and batch == 256 and x_loc.shape[0] == 256
        first = dp.sum_(x_loc[0, 0, :1].clone())          # rank 0 starts at row 0, rank 1 at row 256: disjoint shards
        assert first.item() == 0.0 + 256 * 2
        for _ in range(steps):                            # one collective per step, as the training steps issue
            dp.sum_(torch.ones(1))
        x_small, _, b_small = trn.shard_equal(rows[:7], rows[:7], 256, dp.world, dp.rank)
        assert x_small.shape[0] == 3 and b_small == 3
        ret[rank] = "ok"
    finally:
        dist.destroy_process_group()


def test_data_parallel_semantics_two_ranks():
    world = 2
    port = 29500 + (os.getpid() % 2000)
    with mp.Manager() as mgr:
        ret = mgr.dict()
        mp.spawn(_worker, args=(world, port, ret), nprocs=world, join=True)
        assert dict(ret) == {0: "ok", 1: "ok"}


def test_single_process_is_noop():
    import importlib.util
    spec = importlib.util.spec_from_file_location("dpd_parallel", os.path.join(ROOT, "6g-pa-gan-dpd_amd", "parallel.py"))
    par = importlib.util.module_from_spec(spec); spec.loader.exec_module(par)
    dp = par.DataParallel()
    assert not dp.enabled and dp.world == 1 and dp.shard_rows(10) == (0, 10)
    x = torch.ones(3, requires_grad=True)
    assert dp.global_sum(x) is x


def test_gloo_never_gets_device_tensors(monkeypatch):
    """gloo's device path can stall for good, so a device tensor is reduced through a host copy, whatever the environment says."""
    import importlib.util
    spec = importlib.util.spec_from_file_location("dpd_parallel", os.path.join(ROOT, "6g-pa-gan-dpd_amd", "parallel.py"))
    par = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(par)
    host = torch.ones(3)

    class OnDevice:
        is_cuda = True

        def detach(self):
            return self

        def cpu(self):
            return host

        def copy_(self, t):
            self.got = t
    seen = []
    monkeypatch.setattr(par.dist, "get_backend", lambda group=None: "gloo")
    monkeypatch.setattr(par.dist, "all_reduce", lambda t, op=None, group=None: seen.append(t))
    monkeypatch.setattr(par.torch.cuda, "synchronize", lambda: None)
    for mode in ("0", "1", "2"):
        monkeypatch.setenv("DPD_GLOO_DEVICE_TENSORS", mode)
        t = OnDevice()
        par._all_reduce(t, dist.ReduceOp.SUM)
        assert seen.pop() is host and t.got is host
