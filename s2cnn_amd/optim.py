"""The step that trains a network: AdamW over all its tensors at once, with moments in 32 or 8 bits, and the norm of their gradients.

The reference trains with torch's own optimizers (examples/mnist/run.py:150-153, examples/shrec17/train.py:66), a handful of launches for
every tensor or every dozen of them; its networks have some tens of tensors of which most are small.  Here all tensors of a list are one launch
(some fifty a launch), the clipping of gradients is part of it, and the moments may take a quarter of the memory.
"""
import ctypes
import struct
from array import array
from operator import attrgetter

import torch

from . import _hip

BLOCK = 256                                              # entries that share a factor where moments are held in 8 bits

_dtype, _requires_grad = attrgetter("dtype"), attrgetter("requires_grad")
_contiguous, _device, _numel, _address = torch.Tensor.is_contiguous, torch.Tensor.get_device, torch.Tensor.numel, torch.Tensor.data_ptr
_TENSORS = {torch.Tensor, torch.nn.Parameter}
_CODES = {torch.float32: (2, 32), torch.float16: (2, 16), torch.bfloat16: (4, 16), torch.float8_e4m3fn: (10, 8), torch.uint8: (1, 8)}      # DLPack's
_ROCM = 10
_LISTS = 0x9E3779B97F4A7C15                              # from the seed of one list of a step to the next's, mod 2^64: odd, so that none comes twice
_STEP = struct.Struct("10PqQ6d3i4x")                     # s2cnn_adamw_t


def _check_list(tensors, dtype, device, what):
    """Dense tensors of one type on one device."""
    if set(map(_dtype, tensors)) != {dtype}:
        raise RuntimeError("%s of one type only, %s (got %s)" % (what, dtype, ", ".join(sorted(map(str, set(map(_dtype, tensors)))))))
    if set(map(_device, tensors)) != {device}:
        raise RuntimeError("%s on the current GPU only, cuda:%d; there is no CPU path" % (what, torch.cuda.current_device() if torch.cuda.is_available() else 0))
    if not all(map(_contiguous, tensors)):
        raise RuntimeError("%s have to be contiguous" % what)


def _described(tensors, dtype, device, n=None):
    """(addresses, numbers of entries) of dense tensors of one type on one device, n the numbers that they have to have; None if they are not, or if
    the library cannot ask."""
    lister = _hip.tensor_list()
    if lister is None or not _TENSORS.issuperset(map(type, tensors)):
        return None
    count = len(tensors)
    out = array("Q", bytes(8 * count))
    found = array("q", bytes(8 * count)) if n is None else n
    objects = array("Q", map(id, tensors))
    code, bits = _CODES[dtype]
    rc = lister[0](lister[1], objects.buffer_info()[0], count, code, bits, _ROCM, device, out.buffer_info()[0], found.buffer_info()[0], int(n is not None))
    return (out, found) if rc == 0 else None


def _list(tensors, dtype, device, what, n=None, copy=False):
    """(addresses, numbers of entries, tensors) of dense tensors of one type on one device; n: the numbers that they have to have; copy: others are copied."""
    known = _described(tensors, dtype, device, n)
    if known is not None:
        return (*known, tensors)
    if copy and not all(map(_contiguous, tensors)):
        with torch.no_grad():
            tensors = [t.contiguous() for t in tensors]
    _check_list(tensors, dtype, device, what)                        # says what is wrong, if anything is
    found = array("q", map(_numel, tensors))
    assert n is None or found == n, "%s of other sizes" % what
    return array("Q", map(_address, tensors)), found, tensors


def _at(a):
    return a.buffer_info()[0] if a is not None else 0


def _current_device(tensors):
    t = tensors[0]
    if not t.is_cuda:
        raise RuntimeError("tensors on the GPU only (got one on %s); there is no CPU path" % t.device)
    return torch._C._cuda_getDevice()


def grad_norm(tensors):
    """
    The root of the sum of squares of all entries of a list of tensors: the norm that gradients are clipped by.

    :param tensors: float32, bfloat16 or float16 (also mixed), on the current GPU; copied where they are not contiguous.  Not differentiated: tensors
        that require gradients (parameters, gradients made with create_graph) are taken under torch.no_grad() only
    :return: float32, no axes, on the GPU: nothing waits for it.  Squares are summed in 64 bits and in an order of their own, so that the result is the
        same every time
    """
    tensors = given = list(tensors)
    if not tensors:
        return torch.zeros((), device="cuda")
    device, count, dtype = _current_device(tensors), len(tensors), tensors[0].dtype
    known = _described(tensors, dtype, device) if dtype in _hip.FLOATS else None
    if known is not None:
        addresses, n = known
        kinds = array("i", [_hip.FLOATS[dtype]]) * count
    else:                                                # of several types, or not all dense
        dtypes = set(map(_dtype, tensors))
        if not dtypes <= _hip.FLOATS.keys():
            raise RuntimeError("tensors of float32, bfloat16 or float16 only (got %s)" % ", ".join(sorted(map(str, dtypes))))
        if set(map(_device, tensors)) != {device}:
            raise RuntimeError("tensors on the current GPU only, cuda:%d; there is no CPU path" % device)
        with torch.no_grad():
            tensors = [t.contiguous() for t in tensors]
        addresses, n = array("Q", map(_address, tensors)), array("q", map(_numel, tensors))
        kinds = array("i", [_hip.FLOATS[d] for d in map(_dtype, tensors)])
    out = torch.empty((), dtype=torch.float32, device=tensors[0].device)
    nbytes = _hip.lib().s2cnn_grad_norm_workspace(_at(n), _at(kinds), count)
    ws = _hip.workspace(nbytes, out.device)
    _hip.call("s2cnn_grad_norm", _at(addresses), _at(n), _at(kinds), count, out.data_ptr(), ws.data_ptr(), nbytes, _hip.stream_ptr())
    # looked for while the kernels run: 4 us of the host's time for a hundred tensors
    assert not (torch.is_grad_enabled() and any(map(_requires_grad, given))), "the norm is not differentiated: torch.no_grad() around it"
    assert not _hip.have_tangents(*given), "the norm is not differentiated"
    return out


def _states(first, second, scales, n, device):
    """Addresses of the moments, in 32 bits (no scales) or 8, of tensors of n entries each."""
    assert len(first) == len(second) == len(n) and (scales is None or len(scales) == len(n))
    one = _list(first, torch.float32 if scales is None else torch.float8_e4m3fn, device, "first moments", n)[0]
    two = _list(second, torch.float32 if scales is None else torch.uint8, device, "second moments", n)[0]
    if scales is None:
        return one, two, None
    return one, two, _list(scales, torch.float32, device, "scales", array("q", [2 * ((x + BLOCK - 1) // BLOCK) for x in n]))[0]


def adamw_step(params, grads, first, second, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, masters=None, scales=None, norm=None,
               max_norm=None, seed=0):
    """
    One step of AdamW on a list of tensors, in place:
    m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2, p = p - lr weight_decay p - lr (m / (1 - b1^step)) / (sqrt(v / (1 - b2^step)) + eps).
    An infinite p stays what it is.

    :param params, grads: tensors of one type (float32, bfloat16 or float16) on the current GPU, as many entries each; parameters contiguous.  No tensor that
        is written (all but the gradients) stands twice in the lists, and no two overlap
    :param first, second: the moments m and v, as many entries as the parameters: float32, or with scales float8_e4m3fn and uint8
    :param step: which step it is, from 1 on: an int, or an int64 tensor of one element on the GPU that is read when the kernels run
    :param lr: a number, or a float32 tensor of one element on the GPU
    :param eps: >= 1e-30
    :param masters: float32 copies of 16-bit parameters, or None: the step is made there, and the parameters are their roundings.  Where a parameter
        is not (the program has set it since), the parameter counts
    :param scales: [ceil(n / 256), 2] float32 for each tensor of n entries: the moments are held in 8 bits, with a factor of each for every
        256 entries, and rounded at random so that their means are right (include/s2cnn_hip.h has the codes; `adamw_states` gives their values).  Zeros
        in all three are moments of zero.  An infinite gradient, or one that is no number, makes all of its 256 entries' moments such
    :param norm, max_norm: gradients are multiplied by min(1, max_norm / norm), norm as `grad_norm` gives it; both or none.  Where it is infinite or no
        number nothing is written
    :param seed: of the random rounding, an int; equal seeds and steps round equal lists alike
    """
    step_of_list = _prepared(params, grads, first, second, step, lr, betas, eps, weight_decay, masters, scales, norm, max_norm, seed)
    if step_of_list is not None:
        _launch(step_of_list)


def _prepared(params, grads, first, second, step, lr, betas, eps, weight_decay, masters, scales, norm, max_norm, seed):
    """`adamw_step`'s arguments, checked: (the library's struct, the parameters, what the struct points into), or None where there is nothing to do."""
    params, grads, first, second = list(params), list(grads), list(first), list(second)
    masters, scales = (list(t) if t is not None else None for t in (masters, scales))
    assert len(params) == len(grads)
    assert 0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0 and 1e-30 <= eps < 1e30 and 0.0 <= weight_decay < 1e30
    assert torch.is_tensor(lr) or 0.0 <= lr < 1e30
    assert isinstance(seed, int)
    assert step.numel() == 1 if torch.is_tensor(step) else isinstance(step, int) and step >= 1
    assert not torch.is_tensor(lr) or lr.numel() == 1
    assert (norm is None) == (max_norm is None)
    if norm is not None:
        assert norm.numel() == 1 and 0.0 < max_norm < 1e38
    if not params:
        assert not first and not second and not masters and not scales
        return None
    dtype, device = params[0].dtype, _current_device(params)
    if dtype not in _hip.FLOATS:
        raise RuntimeError("float32, bfloat16 or float16 parameters only (got %s)" % dtype)
    p, n, _ = _list(params, dtype, device, "parameters")
    assert len(set(p)) == len(n) or len(set(p) - {0}) == len(n) - n.count(0), "a parameter twice in the list"
    g, _, grads = _list(grads, dtype, device, "gradients", n, copy=True)
    one, two, factors = _states(first, second, scales, n, device)
    copies = None
    if masters is not None:
        assert dtype != torch.float32, "float32 parameters have no masters"
        assert len(masters) == len(n)
        copies = _list(masters, torch.float32, device, "masters", n)[0]
    if torch.is_tensor(step):
        _hip.require_gpu_of(torch.int64, step)
    if torch.is_tensor(lr):
        _hip.require_gpu_of(torch.float32, lr)
    _hip.require_gpu_of(torch.float32, norm)

    step_at, step = (step.data_ptr(), 0) if torch.is_tensor(step) else (0, step)
    lr_at, lr = (lr.data_ptr(), 0.0) if torch.is_tensor(lr) else (0, lr)
    a = _hip.AdamW.from_buffer_copy(_STEP.pack(
        _at(p), _at(g), _at(one), _at(two), _at(factors), _at(copies), _at(n), lr_at, 0 if norm is None else norm.data_ptr(), step_at, step,
        seed & 0xFFFFFFFFFFFFFFFF, lr, *betas, eps, weight_decay, max_norm or 0.0, len(n), _hip.FLOATS[dtype], 32 if scales is None else 8))
    return a, params, (p, g, one, two, factors, copies, n, grads, first, second, masters, scales)


def _launch(prepared):
    _hip.call("s2cnn_adamw_step", ctypes.byref(prepared[0]), _hip.stream_ptr())
    torch.autograd.graph.increment_version(prepared[1])              # as other operations in place do


def adamw_states(first, second, scales):
    """
    The moments that are held in 8 bits, in float32: (list of first moments, list of second moments), of the shapes of the arguments.

    :param first, second, scales: as for `adamw_step`
    """
    first, second, scales = list(first), list(second), list(scales)
    if not first:
        assert not second and not scales
        return [], []
    device = _current_device(first)
    n = array("q", map(_numel, first))
    lists = _states(first, second, scales, n, device)
    out = [[torch.empty(t.shape, dtype=torch.float32, device=t.device) for t in first] for _ in range(2)]
    lists += tuple(array("Q", map(_address, t)) for t in out)
    _hip.call("s2cnn_adamw_states", *map(_at, lists), _at(n), len(n), _hip.stream_ptr())
    return tuple(out)


class AdamW(torch.optim.Optimizer):
    """
    torch.optim.AdamW's steps by `adamw_step`: one launch for some fifty tensors, which a HIP graph may hold.

    :param params: parameters or groups of them, float32, bfloat16 or float16, contiguous, on one GPU.  A group may have its own lr, betas, eps,
        weight_decay, state_bits and masters (the last two count at a parameter's first step)
    :param lr: a number, or a float32 tensor of one element on the GPU, which a captured step reads at every replay
    :param state_bits: 32, or 8: two bytes a parameter for the moments instead of eight, and a thirty-second of one for their factors
    :param masters: float32 copies of 16-bit parameters, in which small steps add up.  The program may set the parameters at any time (load a
        state dict): where they are not their masters' roundings, they count
    :param max_norm: gradients are clipped to this norm, of all groups together (`self.norm` is the norm of the last step, before it): multiplied by
        min(1, max_norm / norm), where torch's clipping adds 1e-6 to the norm; a step whose norm is infinite or no number is left out and not
        counted.  None: neither
    :param seed: of the random rounding of moments in 8 bits; ranks of a job that hold the same parameters need the same.  Lists of a step (groups, types,
        counts) take random numbers of their own each

    Steps are counted on the device, for every parameter those that it had a gradient in; a step that raises is not made for any.  State dicts hold the
    moments as they are; max_norm and seed are the program's to keep.  A step that a graph captures needs the moments to exist, and the same parameters
    to have gradients as before: make one before.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, masters=True, max_norm=None, seed=0):
        assert max_norm is None or 0.0 < max_norm < 1e38
        assert isinstance(seed, int)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, masters=masters))
        self.max_norm, self.seed, self.norm = max_norm, seed, None

    def __getstate__(self):
        return {**super().__getstate__(), "max_norm": self.max_norm, "seed": self.seed, "norm": self.norm}

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        try:
            self._check_group(self.param_groups[-1])
        except Exception:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_group(group):
        assert group["state_bits"] in (8, 32)
        assert 0.0 <= group["betas"][0] < 1.0 and 0.0 <= group["betas"][1] < 1.0 and 1e-30 <= group["eps"] < 1e30 and 0.0 <= group["weight_decay"] < 1e30
        assert torch.is_tensor(group["lr"]) and group["lr"].numel() == 1 or 0.0 <= group["lr"] < 1e30
        for p in group["params"]:
            if p.dtype not in _hip.FLOATS:
                raise RuntimeError("float32, bfloat16 or float16 parameters only (got %s)" % p.dtype)

    @staticmethod
    def _no_capture(what):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW %s in a captured step, which every replay would do again: make a step before the capture" % what)

    def _new_state(self, p, group, count):
        state = {"step": count}
        if group["state_bits"] == 8:
            state["first"] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
            state["second"] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device)
            state["scales"] = torch.zeros(-(-p.numel() // BLOCK), 2, device=p.device)
        else:
            state["first"], state["second"] = (torch.zeros(p.shape, device=p.device) for _ in range(2))
        if group["masters"] and p.dtype != torch.float32:
            state["master"] = p.detach().float().contiguous()
        return state

    def _lists(self, group):
        """[(count of steps, parameters, their states)] of a group's parameters that have a gradient, those of equal counts together, by type.  Parameters
        that were stepped together so far share one count."""
        members, stepped, fresh = {}, {}, {}
        for p in group["params"]:
            state = self.state.get(p)
            if state:
                members[id(state["step"])] = members.get(id(state["step"]), 0) + 1
            if p.grad is None:
                continue
            if p.grad.is_sparse:
                raise RuntimeError("AdamW takes no sparse gradients")
            if not state:
                self._no_capture("begins with a parameter")
                key = p.device
                if key not in fresh:
                    fresh[key] = torch.zeros(1, dtype=torch.int64, device=p.device)
                state = self.state[p] = self._new_state(p, group, fresh[key])
                members[id(state["step"])] = members.get(id(state["step"]), 0) + 1
            params, states = stepped.setdefault(id(state["step"]), ([], []))
            params.append(p)
            states.append(state)
        lists = []
        for key, (params, states) in stepped.items():
            count = states[0]["step"]
            if len(params) < members[key]:                               # some of them are left out of this step: from here on they count apart
                self._no_capture("leaves a parameter out for the first time")
                count = count.clone()
                for state in states:
                    state["step"] = count
            lists.append((count, params, states))
        return lists

    @torch.no_grad()
    def step(self, closure=None):
        """One step on all parameters that have a gradient; the loss of `closure`, if there is one."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        finite = None
        if self.max_norm is not None:
            self.norm = grad_norm([p.grad for group in self.param_groups for p in group["params"] if p.grad is not None])
            finite = torch.isfinite(self.norm)
        steps, counts = [], []                                           # all lists are checked before the first is stepped or counted
        for group in self.param_groups:
            for count, params, states in self._lists(group):
                counts.append(count)
                kinds = {}                                               # what is held of a parameter was chosen when it was first stepped
                for p, state in zip(params, states):
                    some, held = kinds.setdefault((p.dtype, "master" in state, "scales" in state), ([], []))
                    some.append(p)
                    held.append(state)
                for (_, masters, scales), (some, held) in kinds.items():
                    steps.append(_prepared(some, [p.grad for p in some], [s["first"] for s in held], [s["second"] for s in held], count, group["lr"],
                                           group["betas"], group["eps"], group["weight_decay"], [s["master"] for s in held] if masters else None,
                                           [s["scales"] for s in held] if scales else None, self.norm if finite is not None else None,
                                           self.max_norm, self.seed + len(steps) * _LISTS))
        for count in counts:
            count.add_(1 if finite is None else finite)
        for prepared in steps:
            _launch(prepared)
        return loss

    def moments(self, p):
        """(first, second) moments of a parameter in float32, whatever they are held in; None before its first step."""
        state = self.state[p] if p in self.state else None
        if not state:
            return None
        if "scales" not in state:
            return state["first"], state["second"]
        (first,), (second,) = adamw_states([state["first"]], [state["second"]], [state["scales"]])
        return first, second

    def load_state_dict(self, state_dict):
        """States keep their types (torch's own method takes them to the parameters')."""
        loaded = {}
        # behind the program's hooks before the loading, which may give another dict, and in front of those after it
        hooks = [self.register_load_state_dict_pre_hook(lambda _, seen: loaded.update(seen)),
                 self.register_load_state_dict_post_hook(lambda _: self._restore(loaded), prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _restore(self, state_dict):
        for group, from_group in zip(self.param_groups, state_dict["param_groups"]):
            if torch.is_tensor(group["lr"]):
                group["lr"] = group["lr"].to(group["params"][0].device)
            counts = {}                                              # parameters of a group that had as many steps go on together
            for i, p in zip(from_group["params"], group["params"]):
                if i in state_dict["state"]:
                    state = {k: t.detach().to(p.device, copy=True) for k, t in state_dict["state"][i].items()}
                    state["step"] = counts.setdefault((int(state["step"]), p.device), state["step"])
                    self.state[p] = state
