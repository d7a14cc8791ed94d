"""Optimiser factories with the call shape of libs/lasagne_libs/updates.py.  The reference's updaters
take symbolic gradients and return (updates OrderedDict, opt_params_dict); here the "updates" object
is an `Update` whose `.apply(network)` runs the fused HIP optimiser kernel on the network's flat
parameter / gradient buffers, and opt_params_dict exposes the same keys ('t_prev', and for Adam
'm_prev' / 'v_prev').

`adam` (libs/lasagne_libs/updates.py:534-618) is what every hot-path script passes
(scripts/exp_deep_lstm2.py:17,85); the scripts around models/gating_hyper_nets.py pick
`eval(args.updater)` among momentum / adam / adamax / nesterov_momentum and clip with
`total_norm_constraint` (scripts/dln/ted/exp_prj_lstm_dln.py:17,135-148).  All of them run as the one
elementwise HIP kernel asr_opt_step; the state tensors are flat, like the parameters.
"""
import copy
from collections import OrderedDict
from collections.abc import Iterable

import numpy as np
import torch

from . import ops


class SharedScalar(object):
    """Minimal stand-in for `theano.shared(floatX(x))`: .get_value() / .set_value()."""
    def __init__(self, value, name=None):
        self.value = np.float32(value); self.name = name

    def get_value(self):
        return self.value

    def set_value(self, v):
        self.value = np.float32(v)


class Update(object):
    def apply(self, network, want_sqrt=True):
        raise NotImplementedError


class AdamUpdate(Update):
    def __init__(self, learning_rate, beta1, beta2, epsilon, t_prev):
        self.learning_rate = learning_rate
        self.beta1, self.beta2, self.epsilon = beta1, beta2, epsilon
        self.t_prev = t_prev

    def _lr(self):
        lr = self.learning_rate
        return float(lr.get_value()) if hasattr(lr, 'get_value') else float(lr)

    def apply(self, network, want_sqrt=True):
        network.t_prev = int(round(float(self.t_prev.get_value())))
        norm = network.adam_update(self._lr(), self.beta1, self.beta2, self.epsilon, want_sqrt=want_sqrt)
        self.t_prev.set_value(network.t_prev)
        return norm


def adam(loss_or_grads=None, params=None, learning_rate=0.001, beta1=0.9, beta2=0.999, epsilon=1e-8,
         load_params_dict=None):
    opt_params_dict = OrderedDict()
    t0 = 0.0
    if load_params_dict:
        t0 = float(np.asarray(load_params_dict['t_prev']))
    t_prev = SharedScalar(t0, 't_prev')
    opt_params_dict['t_prev'] = t_prev
    if isinstance(loss_or_grads, ClippedGrads):        # adam behind total_norm_constraint
        return OptUpdate(7, learning_rate, beta1, beta2, epsilon, loss_or_grads, t_prev, beta1), opt_params_dict
    return AdamUpdate(learning_rate, beta1, beta2, epsilon, t_prev), opt_params_dict


class ClippedGrads(object):
    """What total_norm_constraint(..., return_norm=True)[0] stands for here: "the network's gradients,
    scaled so that their global norm is at most max_norm" -- applied inside the optimiser kernel."""
    def __init__(self, max_norm, epsilon):
        self.max_norm = float(max_norm); self.epsilon = float(epsilon)

    def __iter__(self):
        raise TypeError("these stand for the network's own gradients, which its updater scales; a list of gradients is scaled by "
                        "itself if it holds float32, bfloat16 or float16 tensors of one GPU (and None)")


class NormHandle(object):
    """Second return value of total_norm_constraint(return_norm=True): filled by the next update."""
    value = None


class ListNorm(torch.Tensor):
    """The same for a list that has been clipped: the norm as a (1,) tensor on the list's GPU, and its .value read from there."""
    __torch_function__ = torch._C._disabled_torch_function_impl

    @property
    def value(self):
        return self.item()

    def __reduce_ex__(self, protocol):                 # copied and saved as the plain tensor that it is otherwise
        return self.as_subclass(torch.Tensor).__reduce_ex__(protocol)

    def __deepcopy__(self, memo):
        return copy.deepcopy(self.as_subclass(torch.Tensor), memo)


class ScaledGrads(list, ClippedGrads):
    """The scaled tensors of a list.  An updater works on its network's own gradients alone: given this, as the reference's scripts
    do, it takes and keeps how those are to be clipped (`own`), by their own norm, and leaves the tensors to the caller."""
    def __init__(self, tensors, max_norm, epsilon):
        list.__init__(self, tensors)
        self.own = ClippedGrads(max_norm, epsilon)

    max_norm = property(lambda self: self.own.max_norm, lambda self, v: setattr(self.own, 'max_norm', v))
    epsilon = property(lambda self: self.own.epsilon, lambda self, v: setattr(self.own, 'epsilon', v))


def total_norm_constraint(tensor_vars=None, max_norm=0.0, epsilon=1e-7, return_norm=False):
    """libs/lasagne_libs/updates.py:781-855 (lasagne.updates.total_norm_constraint).  GPU tensors in a list or any other iterable
    (gradients held outside a network's flat buffer, such as those of asr_amd.ops.selective_scan_bwd) are clipped here and now: the
    list of the scaled tensors is returned (None, a parameter without a gradient, stays None), with the norm as a (1,) tensor if
    return_norm (its .value is the number).  Anything else stands for the network's own gradients, which the optimiser kernel
    scales when it reads them: lists that ops.clip_list refuses too (other types, tensors on several devices, a max_norm or an
    epsilon below zero)."""
    cg = ClippedGrads(max_norm, epsilon)
    if (isinstance(tensor_vars, Iterable) and not isinstance(tensor_vars, (torch.Tensor, np.ndarray, str, dict))
            and type(tensor_vars) is not ClippedGrads):
        every = list(tensor_vars)
        there = [t for t in every if t is not None]
        if all(isinstance(t, torch.Tensor) for t in there) and any(t.is_cuda for t in there):
            try:
                scaled, norm = ops.clip_list(there, cg.max_norm, cg.epsilon)
            except ValueError:                             # refused before anything was launched
                pass
            else:
                if len(there) < len(every):
                    left = iter(scaled)
                    scaled = [None if t is None else next(left) for t in every]
                scaled = ScaledGrads(scaled, max_norm, epsilon)
                return (scaled, norm.as_subclass(ListNorm)) if return_norm else scaled
    return (cg, NormHandle()) if return_norm else cg


class OptUpdate(Update):
    """sgd / momentum / nesterov / adagrad / rmsprop / adadelta / adamax on asr_opt_step."""
    def __init__(self, kind, learning_rate, h1, h2, eps, grads, t_prev=None, beta1=None):
        self.kind = kind; self.learning_rate = learning_rate
        self.h1, self.h2, self.eps = h1, h2, eps
        self.t_prev = t_prev; self.beta1 = beta1
        self.clip = grads.own if isinstance(grads, ScaledGrads) else grads if isinstance(grads, ClippedGrads) else None

    def _lr(self):
        lr = self.learning_rate
        return float(lr.get_value()) if hasattr(lr, 'get_value') else float(lr)

    def apply(self, network, want_sqrt=True):
        lr = self._lr()
        if self.kind == 6:                       # adamax: a_t = lr / (1 - beta1^t), :662-664
            t = int(round(float(self.t_prev.get_value()))) + 1
            self.t_prev.set_value(t)
            lr = lr / (1.0 - self.beta1 ** t)
        elif self.kind == 7:                     # adam with gradient clipping
            t = int(round(float(self.t_prev.get_value()))) + 1
            self.t_prev.set_value(t)
            network.t_prev = t
            lr = lr * np.sqrt(1.0 - self.h2 ** t) / (1.0 - self.h1 ** t)
        mg = self.clip.max_norm if self.clip else 0.0
        ne = self.clip.epsilon if self.clip else 1e-7
        return network.opt_update(self.kind, lr, self.h1, self.h2, self.eps, mg, ne, want_sqrt=want_sqrt)


def _mk(kind, grads, learning_rate, h1=0.0, h2=0.0, eps=0.0, with_t=False, load_params_dict=None):
    d = OrderedDict()
    t_prev = None
    if with_t:
        t_prev = SharedScalar(float(np.asarray(load_params_dict['t_prev'])) if load_params_dict else 0.0, 't_prev')
        d['t_prev'] = t_prev
    return OptUpdate(kind, learning_rate, h1, h2, eps, grads, t_prev, h1 if with_t else None), d


def sgd(loss_or_grads=None, params=None, learning_rate=0.0, load_params_dict=None):
    """:64-92."""
    return _mk(0, loss_or_grads, learning_rate)


def momentum(loss_or_grads=None, params=None, learning_rate=0.0, momentum=0.9, load_params_dict=None):
    """:152-188 (sgd + apply_momentum :95-149)."""
    return _mk(1, loss_or_grads, learning_rate, momentum)


def nesterov_momentum(loss_or_grads=None, params=None, learning_rate=0.0, momentum=0.9, load_params_dict=None):
    """:254-295 (sgd + apply_nesterov_momentum :191-251)."""
    return _mk(2, loss_or_grads, learning_rate, momentum)


def adagrad(loss_or_grads=None, params=None, learning_rate=1.0, epsilon=1e-6, load_params_dict=None):
    """:298-363."""
    return _mk(3, loss_or_grads, learning_rate, eps=epsilon)


def rmsprop(loss_or_grads=None, params=None, learning_rate=1.0, rho=0.9, epsilon=1e-6, load_params_dict=None):
    """:366-433."""
    return _mk(4, loss_or_grads, learning_rate, rho, eps=epsilon)


def adadelta(loss_or_grads=None, params=None, learning_rate=1.0, rho=0.95, epsilon=1e-6, load_params_dict=None):
    """:436-531."""
    return _mk(5, loss_or_grads, learning_rate, rho, eps=epsilon)


def adamax(loss_or_grads=None, params=None, learning_rate=0.002, beta1=0.9, beta2=0.999, epsilon=1e-8,
           load_params_dict=None):
    """:621-698."""
    return _mk(6, loss_or_grads, learning_rate, beta1, beta2, epsilon, with_t=True, load_params_dict=load_params_dict)
