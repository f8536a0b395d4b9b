"""GraphSAGE with RMS norm and residual layers on several ranks: the norms' gradients travel with
those of their layers."""
import json
import os
import socket
import subprocess
import sys

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp
import torch.nn.functional as F

from grappa_b200.block import Block
from grappa_b200.models import SAGE

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _free_port():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    p = s.getsockname()[1]
    s.close()
    return p


def _model():
    torch.manual_seed(0)
    return SAGE(6, 8, 3, 4, F.silu, 0.0, norm="rms", residual=True)


def _gradient(model, seed):
    g = torch.Generator().manual_seed(seed)
    n = 25
    indptr = torch.zeros(n + 1, dtype=torch.int64)
    indptr[1:] = torch.cumsum(torch.randint(1, 4, (n,), generator=g), 0)
    b = Block(indptr, torch.randint(0, n, (int(indptr[-1]),), generator=g), torch.arange(n), n, n)
    x, y = torch.randn(n, 6, generator=g), torch.randint(0, 3, (n,), generator=g)
    F.cross_entropy(model([b] * 4, x), y).backward()
    return {k: p.grad.clone() for k, p in model.named_parameters()}


def _rank(rank, port, q):
    from grappa_b200.grad import coverage_all_reduce

    torch.set_num_threads(2)
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=2)
    m = _model()
    _gradient(m, rank)
    coverage_all_reduce(list(m.parameters()), 0.5 + 0.25 * rank, 2)
    q.put((rank, {k: p.grad.numpy().copy() for k, p in m.named_parameters()}))
    dist.barrier()
    dist.destroy_process_group()


def test_two_ranks_reduce_every_gradient():
    ctx = mp.get_context("spawn")
    q, port = ctx.Queue(), _free_port()
    ps = [ctx.Process(target=_rank, args=(r, port, q)) for r in range(2)]
    for p in ps:
        p.start()
    got = dict(q.get(timeout=120) for _ in ps)
    for p in ps:
        p.join(timeout=60)
    own = [_gradient(_model(), r) for r in range(2)]
    assert any(k.startswith("norms") for k in own[0])
    for k in own[0]:
        want = (0.5 * own[0][k] + 0.75 * own[1][k]) / 2
        assert float(want.abs().max()) > 0
        for r in range(2):
            # two products and a sum in fp32
            torch.testing.assert_close(torch.from_numpy(got[r][k]), want, rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("layers,hidden", [(2, 16), (4, 16), (5, 100)])
def test_a_bucket_holds_a_layer_with_its_norm(layers, hidden):
    m = SAGE(10, hidden, 7, layers, norm="rms", residual=True)
    buckets = m.layer_buckets(layers)
    assert buckets[0][0] == 0 and buckets[-1][1] == m.num_flat
    assert all(a[1] == b[0] for a, b in zip(buckets, buckets[1:]))
    for i, (lo, hi) in enumerate(buckets):
        names = [n for n, s in m._segments.items() if lo <= s.offset and s.offset + s.numel <= hi]
        assert sorted(names) == sorted([f"layers.{i}.W", f"layers.{i}.b"] + ([f"layers.{i}.norm"] if i else []))


def test_command_line_on_two_ranks(tmp_path):
    from grappa_b200.dataset import partition

    d = tmp_path
    assert partition.main(["generate", "--graph_name", "tiny", "--out", str(d / "t10n" / "tiny")]) == 0
    assert partition.main(["seq", "--src_path", str(d / "t10n" / "tiny"), "--dest_path", str(d), "--graph_name", "tiny",
                           "--n_part", "2"]) == 0
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node", "2", "--master-addr",
           "127.0.0.1", "--master-port", str(_free_port()), "-m", "grappa_b200.train.t10n_train", "--data_path", str(d),
           "--graph_name", "tiny", "--part_method", "hash", "--n_part", "2", "--model", "sage", "--num_hidden", "16",
           "--num_layers", "3", "--fan_out", "3,3,3", "--num_epochs", "2", "--batch_size", "256", "--batch_size_eval",
           "1000", "--eval_every", "2", "--repart_every", "2", "--num_gpus", "-1", "--backend", "gloo", "--tag_id", "r",
           "--close_dd", "--norm", "rms", "--residual", "--activation", "silu", "--dropout", "0.2", "--metrics_jsonl",
           str(tmp_path / "m_{rank}.jsonl")]
    r = subprocess.run(cmd, cwd=ROOT, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, (r.stdout + r.stderr)[-4000:]
    recs = [json.loads(line) for line in open(tmp_path / "m_0.jsonl")]
    assert recs
