"""The norm of all gradients of a model together, and clipping by it.

    norm = (sum |g|^p over every element)^(1/p),  p = 1, 2 or infinity
    g    = g * min(1, max_norm / (norm + 1e-6))

Both run on the device without a host read: the norm comes back as an fp32 tensor, from 64-bit
sums in a fixed order (the same bits on every run), and the clipping decides there whether there
is anything to scale.
"""

from array import array
from operator import attrgetter

import torch

from . import _lib
from .objective_ops import refuse_tangents

_ORDERS = {1.0: 1, 2.0: 2, float("inf"): 0}
_Tensor = torch.Tensor
_dtype_of = attrgetter("dtype")
_grad_of = attrgetter("grad")


def _order(what, norm_type):
    try:
        return _ORDERS[float(norm_type)]
    except KeyError:
        raise ValueError(f"{what}: norm_type is 1, 2 or inf, got {norm_type}") from None


def _fills_its_memory(t):
    """True when the elements of a strided tensor are one run of memory in some order, each
    once (a transposed matrix, say): the norm and the scaling do not care about the order."""
    run = 1
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n > 1),
                               key=lambda d: d[1]):
        if stride != run:
            return False
        run *= size
    return True


def _table(what, tensors):
    """(device, addresses, sizes, dtype tags) as the C-ABI takes them, and the tensors that were
    replaced by contiguous copies, [(tensor, copy)]. Each property of a tensor costs about 60 ns
    to ask for and a model has hundreds of them, so each is asked for once."""
    try:
        devices = set(map(_Tensor.get_device, tensors))
        contiguous = all(map(_Tensor.is_contiguous, tensors))
        copies = []
        if not contiguous:
            tensors = list(tensors)
            for i, t in enumerate(tensors):
                if not t.is_contiguous() and not _fills_its_memory(t):
                    copies.append((t, t.contiguous()))
                    tensors[i] = copies[-1][1]
        ptrs = array("Q", map(_Tensor.data_ptr, tensors))
    except (RuntimeError, NotImplementedError) as e:
        raise TypeError(f"qlora_b200 {what}: dense tensors only ({e})") from e
    if min(devices) < 0:
        raise RuntimeError(f"qlora_b200 {what}: expects CUDA tensors (there is no CPU path)")
    if len(devices) > 1:
        raise ValueError(f"{what}: tensors on several devices ({sorted(devices)})")
    dtypes = list(map(_dtype_of, tensors))
    kinds = set(dtypes)
    tags = bytes([_lib.tag(dtypes[0])]) * len(dtypes) if len(kinds) == 1 else \
        bytes(map(_lib.tag, dtypes))
    return tensors[0].device, ptrs, array("q", map(_Tensor.numel, tensors)), tags, copies


def _run(name, dev, ptrs, sizes, tags, order, max_norm=None):
    n = len(ptrs)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    doubles = _lib.load().qb_grad_norm_workspace(n)
    work = torch.empty(doubles, dtype=torch.float64, device=dev)
    limit = () if max_norm is None else (array("d", [max_norm]),)

    def moved():                     # a kernel timer asks when the norm is known
        once = sum(s * (4 if t == _lib.F32 else 2) for s, t in zip(sizes, tags))
        scaled = limit and not max_norm >= float(seen) + 1e-6
        return 3 * once if scaled else once

    _lib.call_on(dev, name, ptrs.buffer_info()[0], sizes.buffer_info()[0], tags, n, order,
                 *(a.buffer_info()[0] for a in limit), work.data_ptr(), doubles, norm.data_ptr(),
                 kernels=2, work=(moved, 0))
    # the caller may write to the norm it gets
    seen = norm.clone() if limit and _lib.timing() else norm
    return norm


@torch.no_grad()
def grad_norm(tensors, norm_type=2.0):
    """The norm of all elements of the tensors (one, or an iterable; fp32, fp16 and bf16, each its
    own) together: an fp32 tensor on their device, NaN when an element is, 0 without elements
    (on the CPU without a tensor)."""
    order = _order("grad_norm", norm_type)
    tensors = [tensors] if isinstance(tensors, _Tensor) else list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    refuse_tangents("grad_norm", tensors)
    dev, ptrs, sizes, tags, copies = _table("grad_norm", tensors)
    return _run("qb_grad_norm", dev, ptrs, sizes, tags, order)


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Scales the gradients of the parameters (one, or an iterable) in place by
    min(1, max_norm / (norm + 1e-6)) and returns their norm before that, as grad_norm does.
    Parameters without a gradient are left out. An infinite or NaN norm spreads into the
    gradients, unless error_if_nonfinite raises before anything is scaled (a host read).
    Gradients that share memory are refused (those with gaps between their elements are scaled
    through a copy and written back, and not looked at for that)."""
    order = _order("clip_grad_norm_", norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"clip_grad_norm_: max_norm {max_norm} is not a number of at least 0")
    if isinstance(parameters, _Tensor):
        parameters = [parameters]
    grads = [g for g in map(_grad_of, parameters) if g is not None]
    if not grads:
        return torch.tensor(0.0)
    refuse_tangents("clip_grad_norm_", grads)
    dev, ptrs, sizes, tags, copies = _table("clip_grad_norm_", grads)
    for t, _ in copies:
        if 0 in (s for n, s in zip(t.shape, t.stride()) if n > 1):
            raise ValueError("clip_grad_norm_: a gradient's elements share memory (an expanded "
                             "tensor)")
    if error_if_nonfinite:
        norm = _run("qb_grad_norm", dev, ptrs, sizes, tags, order)
        if not torch.isfinite(norm):
            raise RuntimeError(f"clip_grad_norm_: the gradients' norm is {norm.item()}")
    norm = _run("qb_grad_clip", dev, ptrs, sizes, tags, order, max_norm)
    for t, c in copies:
        t.copy_(c)
    torch.autograd.graph.increment_version(grads)
    return norm
