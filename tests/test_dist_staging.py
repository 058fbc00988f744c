"""gloo is handed host memory only: with the collectives replaced by recorders and CUDA tensors without storage (FakeTensorMode, no GPU
needed), everything the helpers hand over lies on the host and every result comes back on the device."""
import types

import pytest
import torch
import torch.distributed as dist
from torch._subclasses.fake_tensor import FakeTensorMode


class Op:
    def __init__(self, op, tensor, peer, group=None):
        self.tensor = tensor


class Done:
    def wait(self):
        pass


@pytest.fixture
def handed(monkeypatch):
    """[device type of every tensor a collective got], as rank 0 of 2."""
    seen = []
    def record(*tensors):
        seen.extend(t.device.type for t in tensors)
    monkeypatch.setattr(dist, 'is_initialized', lambda: True)
    monkeypatch.setattr(dist, 'get_world_size', lambda group=None: 2)
    monkeypatch.setattr(dist, 'get_rank', lambda group=None: 0)
    monkeypatch.setattr(dist, 'all_gather_into_tensor', lambda out, x, group=None: record(out, x))
    monkeypatch.setattr(dist, 'all_reduce', lambda t, op=None, group=None: record(t))
    monkeypatch.setattr(dist, 'reduce_scatter_tensor', lambda out, x, group=None: record(out, x))
    monkeypatch.setattr(dist, 'P2POp', Op)
    monkeypatch.setattr(dist, 'batch_isend_irecv', lambda ops: [record(o.tensor) or Done() for o in ops])
    return seen


@pytest.mark.parametrize("backend,where", [('gloo', 'cpu'), ('nccl', 'cuda')])
@pytest.mark.parametrize("direct", [False, True])
def test_gather_views(handed, monkeypatch, backend, where, direct):
    from gendr_amd.dist import _GatherViews                      # (autograd itself needs a device for CUDA tensors)
    monkeypatch.setattr(dist, 'get_backend', lambda group=None: backend)
    ctx = types.SimpleNamespace()
    with FakeTensorMode():
        views = _GatherViews.forward(ctx, torch.empty(3, 4, 5, device='cuda'), None, True, direct)
        assert views.device.type == 'cuda' and views.shape == (6, 4, 5)
        forward = len(handed)
        grad = _GatherViews.backward(ctx, torch.empty(6, 5, 4, device='cuda').transpose(1, 2))[0]
        assert grad.device.type == 'cuda' and grad.shape == (3, 4, 5)
    assert forward >= 2 and len(handed) > forward and set(handed) == {where}, handed


@pytest.mark.parametrize("backend,where", [('gloo', 'cpu'), ('nccl', 'cuda')])
@pytest.mark.parametrize("leaf", [False, True])
def test_sum_over_ranks(handed, monkeypatch, backend, where, leaf):
    from gendr_amd.dist import sum_over_ranks
    monkeypatch.setattr(dist, 'get_backend', lambda group=None: backend)
    with FakeTensorMode():
        t = torch.empty(7, 3, device='cuda', requires_grad=leaf)
        assert sum_over_ranks(t) is t and t.device.type == 'cuda'
    assert handed == [where]


def test_bench_reduces_its_time_on_the_host():
    """bench.py joins the ranks' elapsed times with one all-reduce: over gloo of a host tensor."""
    import os
    import re
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'bench.py'), encoding='utf-8').read()
    lines = re.findall(r'torch\.tensor\(\[elapsed\].*', src)
    assert len(lines) == 1 and "'cpu' if stub or dist.get_backend() == 'gloo' else dev" in lines[0], lines
