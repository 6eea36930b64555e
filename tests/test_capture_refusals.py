"""A graph capture of a step with active collectives is refused before anything is launched (one-rank gloo group, no GPU)."""
from types import SimpleNamespace

import pytest
import torch
import torch.distributed as dist

from ha2g_amd import ddp
from ha2g_amd.train import HierarchyTrainer


@pytest.fixture
def one_rank(monkeypatch):
    dist.init_process_group('gloo', store=dist.HashStore(), rank=0, world_size=1)
    monkeypatch.setattr(ddp, 'FORCE_ACTIVE', True)
    yield
    dist.destroy_process_group()


def test_capture_step_refuses_active_collectives(one_rank):
    tr = HierarchyTrainer.__new__(HierarchyTrainer)
    tr.train_iter = lambda *a, **k: pytest.fail('the step ran')
    with pytest.raises(RuntimeError, match='collectives'):
        tr.capture_step(11, None, None, None, None)


@pytest.mark.parametrize('call', (lambda t: ddp.all_reduce_(t), lambda t: ddp.sync_flag_(t), lambda t: ddp.all_gather_([t], t), lambda t: ddp.broadcast_one_(t),
                                  lambda t: ddp.broadcast_([t]), lambda t: ddp.prefetch_max_count(t)))
def test_collectives_refuse_a_capturing_stream(one_rank, monkeypatch, call):
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    with pytest.raises(RuntimeError, match='inside a graph capture'):
        call(SimpleNamespace(is_cuda=True))


def test_collectives_of_host_tensors_run(one_rank):
    t = torch.ones(3)
    ddp.all_reduce_(t)
    ddp.broadcast_one_(t)
    assert torch.equal(t, torch.ones(3))
