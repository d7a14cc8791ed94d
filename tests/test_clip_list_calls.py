"""updates.total_norm_constraint as a call: what it takes for a list of gradients to clip and what for the network's own, what it
returns, and what an updater keeps of it."""
import copy
import io
import pickle
import weakref

import numpy as np
import pytest
import torch

from asr_amd import ops, updates


class OnGpu(torch.Tensor):
    is_cuda = True


def on_gpu(*shape, dtype=torch.float32):
    return torch.ones(*shape, dtype=dtype).as_subclass(OnGpu)


def is_stand_in(tensors, *args):
    """-> the result stands for the network's own gradients, as it does for any argument that is no list of GPU tensors"""
    cg, handle = updates.total_norm_constraint(tensors, *args, return_norm=True)
    assert type(updates.total_norm_constraint(tensors, *args)) is updates.ClippedGrads
    step, _ = updates.adam(cg)
    assert step.kind == 7 and step.clip is cg and cg.max_norm == float(args[0])
    with pytest.raises(TypeError, match='own gradients'):
        list(cg)
    return type(cg) is updates.ClippedGrads and type(handle) is updates.NormHandle


def test_lists_that_cannot_be_clipped_stand_for_the_network_as_before():
    for bad in ([on_gpu(3, dtype=torch.float64)], [on_gpu(3), on_gpu(2, dtype=torch.int64)], (on_gpu(3), torch.ones(2))):
        assert is_stand_in(bad, 1.0)
    for max_norm in (-1.0, np.float32(-2.0)):
        assert is_stand_in([on_gpu(3)], max_norm)
    assert is_stand_in([on_gpu(3)], 1.0, -1e-7)
    for sparse in (torch.eye(3).to_sparse(), torch.eye(3).to_sparse_csr()):
        with pytest.raises(ValueError, match='strided'):
            ops.clip_list([torch.ones(3), sparse], 1.0)


def clip_on_the_cpu(monkeypatch):
    monkeypatch.setattr(ops, 'clip_list', lambda tensors, max_norm, eps: ([t.as_subclass(torch.Tensor) + 1 for t in tensors], torch.full((1,), 2.5)))


def test_norm_of_a_list_has_a_value_like_the_network_s(monkeypatch):
    clip_on_the_cpu(monkeypatch)
    _, handle = updates.total_norm_constraint(None, 1.0, return_norm=True)
    assert handle.value is None
    _, norm = updates.total_norm_constraint([on_gpu(3)], 1.0, return_norm=True)
    assert norm.value == 2.5 and norm.shape == (1,) and type(norm.reshape(()) + 1) is torch.Tensor
    file = io.BytesIO()                                                 # copied and saved like any tensor
    torch.save(norm, file)
    file.seek(0)
    for again in (copy.deepcopy(norm), copy.copy(norm), pickle.loads(pickle.dumps(norm)), torch.load(file, weights_only=True)):
        assert torch.equal(again, torch.full((1,), 2.5))


@pytest.mark.parametrize('kind', [list, tuple, iter, lambda ts: (t for t in ts), lambda ts: dict(enumerate(ts)).values()])
def test_gradients_in_any_iterable_and_parameters_without_one(kind, monkeypatch):
    clip_on_the_cpu(monkeypatch)
    got, norm = updates.total_norm_constraint(kind([None, on_gpu(3), None, on_gpu(2), None]), 1.0, return_norm=True)
    assert type(got) is updates.ScaledGrads and len(got) == 5 and got[0] is got[2] is got[4] is None
    assert torch.equal(got[1], torch.full((3,), 2.0)) and torch.equal(got[3], torch.full((2,), 2.0)) and norm.value == 2.5
    assert type(updates.total_norm_constraint(kind([on_gpu(1)]), 1.0)) is updates.ScaledGrads
    once = updates.ScaledGrads([on_gpu(1)], 1.0, 1e-7)                  # clipped again
    assert torch.equal(updates.total_norm_constraint(once, 1.0)[0], torch.full((1,), 2.0))


def test_an_updater_keeps_no_scaled_tensors():
    """only how its network's gradients are to be clipped, whatever becomes of the list"""
    class Net(object):
        def opt_update(self, kind, lr, h1, h2, eps, max_norm, norm_eps, want_sqrt):
            self.clipped = max_norm, norm_eps
    for updater in (updates.adam, updates.sgd, updates.adamax):
        tensors = [torch.ones(3), torch.ones(2)]
        gone = weakref.ref(tensors[0])
        scaled = updates.ScaledGrads(tensors, 5.0, 1e-6)
        step, _ = updater(scaled, learning_rate=0.1)
        scaled.max_norm = 4.0                                           # what a script sets later counts, as for the network's own
        assert step.clip.max_norm == 4.0 and scaled.max_norm == 4.0 and scaled.epsilon == 1e-6
        del scaled[:]
        net = Net()
        step.apply(net)
        assert net.clipped == (4.0, 1e-6)
        del tensors, scaled
        assert gone() is None


def test_what_holds_no_gpu_tensor_stands_for_the_network_as_before():
    for own in (None, [], [None], (), 'grads', np.zeros(3), torch.zeros(3), on_gpu(3), {'w': on_gpu(3)}, [np.zeros(3)], [torch.zeros(3), None],
                iter([np.zeros(3)]), updates.ClippedGrads(1.0, 1e-7)):
        assert is_stand_in(own, 1.0)


@pytest.mark.gpu
def test_gpu_lists_that_cannot_be_clipped_stand_for_the_network_as_before():
    t = torch.ones(3, device='cuda')
    for bad in ([t.double()], [t, t.long()], [t, torch.ones(2)], [torch.ones(2), t], [t.to_sparse()], [torch.eye(3, device='cuda').to_sparse_csr()]):
        assert is_stand_in(bad, 1.0)
    assert is_stand_in([t], -1.0)


@pytest.mark.gpu
def test_max_norm_is_taken_as_a_number():
    """a numpy scalar or a tensor of one value, as before"""
    t = torch.full((4,), 3.0, device='cuda')
    want = updates.total_norm_constraint([t], 1.5)
    for m in (np.float32(1.5), torch.tensor(1.5), torch.tensor([1.5], device='cuda')):
        got = updates.total_norm_constraint([t], m)
        assert torch.equal(got[0], want[0]) and got.max_norm == 1.5
    _, norm = updates.total_norm_constraint([t], 1.5, return_norm=True)
    assert norm.is_cuda and norm.value == 6.0
