"""The encoder's training example on a GPU."""
import importlib.util
import os
import subprocess
import sys

import pytest
import torch

from mp_util import free_port

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example(name):
    spec = importlib.util.spec_from_file_location(name, os.path.join(ROOT, "examples", name + ".py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_a_batch_stays_until_it_has_been_read():
    """The host runs ahead of a device that takes its time: no later batch may take the place of one that is still to be read."""
    host = [tuple(torch.full((n,), 10 * i + j).pin_memory() for j, n in enumerate((4096, 37, 1))) for i in range(3)]
    seen = []
    for _, batch in zip(range(9), _example("bert_pretrain").device_batches(host, torch.device("cuda"))):
        torch.cuda._sleep(20_000_000)  # about a hundredth of a second
        seen.append([t.clone() for t in batch])
        del batch
    torch.cuda.synchronize()
    for i, batch in enumerate(seen):
        for got, want in zip(batch, host[i % 3]):
            assert torch.equal(got.cpu(), want), i


@pytest.mark.parametrize("options", [[], ["--padded", "--save8"]])
def test_the_encoder_example_runs(options, tmp_path):
    path = tmp_path / "model.pt"
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=1", "--master-addr", "127.0.0.1", "--master-port",
           str(free_port()), os.path.join(ROOT, "examples", "bert_pretrain.py"), "--steps", "7", "--batch", "3", "--seq", "100", "--layers", "1",
           "--checkpoint", str(path), *options]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-3000:]
    assert "step 6: loss" in r.stdout and "tokens/s" in r.stdout and path.exists()
