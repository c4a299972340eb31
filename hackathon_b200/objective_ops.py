"""The post-training ops as PyTorch operators (namespace `qlora_b200`, beside those of ops.py):

    op                      computes                                          backward
    token_logprobs          log-probability of each row's target token, the   token_logprobs_bwd
                            row's entropy, (max, sum) of the row
    token_logprobs_bwd      dlogits
    preference              pairs' loss; rewards and each row's coefficient   preference_bwd
    preference_bwd          dlogp = mask * coefficient * g
    policy                  clipped policy loss + KL; its statistics, the     policy_bwd
                            rows' weights, the unit gradient
    policy_bwd              dlogp = unit gradient * row weight * g

The functions users call (logprobs.py, preference.py, policy.py) check their arguments and bring
them into the layouts these ops read. The kernels of an objective take a few microseconds at the
sizes of a batch, so the host's part decides: the ops are registered with torch.library's
define / impl and an autograd.Function of their own (a preference loss and its gradient took
239 us of host time through torch.library.custom_op and its generated formula and takes 112 now,
69 of them an empty autograd.Function's), and small outputs share one allocation with the
workspace.
"""

import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import NS

F32, F64 = torch.float32, torch.float64
_library = torch.library.Library(NS, "FRAGMENT")
_ops = getattr(torch.ops, NS)
_below_autograd = torch._C._AutoDispatchBelowAutograd
transformed = torch._C._are_functorch_transforms_active
_profiled = torch.autograd._profiler_enabled
_NATIVE = frozenset((torch.Tensor, torch.nn.Parameter, float, int, bool, type(None), torch.dtype))


def _plain(args):
    """A call the dispatcher would hand to the CUDA kernel as it is: no tensor subclass (fake and
    functional tensors are) or symbolic number among the arguments, no mode that wants to see the
    op, no profiler that records it by its name, and no function transform, whose tensors are of
    the plain type and hold no memory."""
    return (_NATIVE.issuperset(map(type, args)) and args[0].is_cuda and not (
        transformed() or _profiled() or torch._C._len_torch_dispatch_stack()))


def _has_tangent(t):
    if not isinstance(t, torch.Tensor):
        return False
    while torch._C._functorch.is_batchedtensor(t):     # a batch's tangent is its base's
        t = torch._C._functorch.get_unwrapped(t)
    return forward_ad.unpack_dual(t).tangent is not None


def refuse_tangents(what, tensors):
    """The kernels have no forward-mode derivative: inside a forward-mode level an input with a
    tangent is refused (a result without its tangent would be a constant)."""
    if forward_ad._current_level >= 0 and any(map(_has_tangent, tensors)):
        raise NotImplementedError(f"{what}: no forward-mode derivative, and an input has a tangent")


def _register(schema, fake, function=None):
    """Registers the decorated function as the CUDA kernel of the op `schema` declares, with its
    fake implementation; `function`: the autograd.Function that runs it when the first argument
    asks for a gradient. Returns what calls the op, with .below for the call below autograd. A
    plain call (_plain) goes to the kernel without the dispatcher, whose boxing of the arguments
    takes 5 to 9 us. Under torch.vmap the dispatcher takes the op to each element; the
    transforms that differentiate refuse an autograd.Function of this kind by name."""
    name = schema[:schema.index("(")]

    def register(kernel):
        _library.define(schema)
        _library.impl(name, kernel, "CUDA")
        torch.library.register_fake(f"{NS}::{name}", fake, lib=_library)
        op = getattr(_ops, name).default

        def below(*args):
            if _plain(args):
                return kernel(*args)
            with _below_autograd():
                return op(*args)

        def autograd(*args):
            refuse_tangents(f"{NS}::{name}", args)
            if torch.is_grad_enabled() and args[0].requires_grad:
                return function.apply(*args)
            return below(*args)

        def call(*args):
            if torch.compiler.is_compiling():
                return op(*args)
            if not _plain(args) or forward_ad._current_level >= 0:
                refuse_tangents(f"{NS}::{name}", args)
                return op(*args)
            if function is not None and torch.is_grad_enabled() and args[0].requires_grad:
                return function.apply(*args)
            return kernel(*args)

        if function is not None:
            _library.impl(name, autograd, "Autograd")
        call.below = below
        return call
    return register


def _need(ok, op, what):
    """The kernels read raw addresses: what an op's caller passes has to be what they read."""
    if not ok:
        raise ValueError(f"qlora_b200::{op}: {what}")


def _fits(t, at, dtype, shape):
    """None, or a contiguous tensor of this dtype and shape on the CUDA device numbered `at`."""
    return t is None or (t.get_device() == at and t.dtype == dtype and t.shape == shape
                         and t.is_contiguous())


def _mask_fits(mask, at, shape):
    return mask is None or _fits(mask, at,
                                 torch.uint8 if mask.dtype == torch.uint8 else torch.bool, shape)


class PreferenceConfig(ctypes.Structure):
    _fields_ = [("beta", ctypes.c_double), ("label_smoothing", ctypes.c_double),
                ("margin", ctypes.c_double), ("denominator", ctypes.c_double),
                ("loss_type", ctypes.c_int32), ("length_normalized", ctypes.c_int32)]


class PolicyConfig(ctypes.Structure):
    _fields_ = [("clip_low", ctypes.c_double), ("clip_high", ctypes.c_double),
                ("delta", ctypes.c_double), ("kl_coef", ctypes.c_double),
                ("denominator", ctypes.c_double), ("reduction", ctypes.c_int32),
                ("pad", ctypes.c_int32)]


# ------------------------------------------------------------------------------------------
# log-probabilities of chosen tokens


def row_layout(logits):
    """(logits, rows, inner, outer stride, inner stride): row r of [..., V] logits starts at
    (r // inner) * outer + (r % inner) * inner stride. Up to two leading dimensions of any
    strides are read in place (a view that drops the last position, an expanded one); the rest
    is copied first."""
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        logits = logits.contiguous()
    if logits.dim() > 3 or logits.dim() == 1:
        logits = logits.reshape(-1, logits.shape[-1])
    if logits.dim() == 2:
        return logits, logits.shape[0], 1, logits.stride(0), 0
    b, s, _ = logits.shape
    if b <= 1 or logits.stride(0) == s * logits.stride(1):
        return logits, b * s, 1, logits.stride(1), 0
    return logits, b * s, max(s, 1), logits.stride(0), logits.stride(1)


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target, temperature, with_entropy):
        logp, entropy, state = token_logprobs.below(logits, target, temperature, with_entropy)
        ctx.save_for_backward(logits, target, state, entropy if with_entropy else None)
        ctx.temperature, ctx.with_entropy = temperature, with_entropy
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*((state,) if with_entropy else (entropy, state)))
        return logp, entropy, state

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logp, g_entropy, _g_state):
        logits, target, state, entropy = ctx.saved_tensors
        if not ctx.with_entropy:
            g_entropy = None
        if g_logp is None and g_entropy is None:
            return None, None, None, None
        return token_logprobs_bwd(logits, target, state, entropy, g_logp, g_entropy,
                                  ctx.temperature), None, None, None


# The second (or third) output of an op is one fp32 buffer: what its backward or the caller reads,
# then, 16-byte aligned, the kernels' workspace. The sizes below are the library's
# qb_*_workspace, written here too because a fake implementation needs them of symbolic sizes.


def _up4(n):
    return (n + 3) // 4 * 4


def logprobs_state(rows, vocab, itemsize):
    """Floats of the third output ((max, sum) of each row, workspace), the workspace's offset."""
    at = _up4(2 * rows)
    batch = 8192 // itemsize                       # elements a CTA reads at a time
    batches = (vocab + batch - 1) // batch
    spans = min(batches, max(1, 1184 // max(rows, 1)))
    return at + (4 * rows * spans if spans > 1 else 0), at


def _token_logprobs_fake(logits, target, temperature, with_entropy):
    size, _ = logprobs_state(target.numel(), logits.shape[-1], logits.element_size())
    return (target.new_empty(target.shape, dtype=F32),
            target.new_empty(target.shape if with_entropy else (0,), dtype=F32),
            target.new_empty((size,), dtype=F32))


@_register("token_logprobs(Tensor logits, Tensor target, float temperature, bool with_entropy) "
           "-> (Tensor, Tensor, Tensor)", _token_logprobs_fake, _TokenLogprobs)
def token_logprobs(logits, target, temperature, with_entropy):
    _need(target.get_device() == logits.get_device() and target.dtype == torch.int64
          and target.shape == logits.shape[:-1], "token_logprobs",
          "target is an int64 tensor of the logits' leading shape on their device")
    z, rows, inner, so, si = row_layout(logits)
    vocab, dev = logits.shape[-1], logits.device
    logp = torch.empty(target.shape, dtype=F32, device=dev)
    entropy = torch.empty(target.shape if with_entropy else (0,), dtype=F32, device=dev)
    size, at = logprobs_state(rows, vocab, z.element_size())
    state = torch.empty(size, dtype=F32, device=dev)
    if rows:
        tgt = target.contiguous()
        _lib.call_on(dev, "qb_token_logprobs", z.data_ptr(), _lib.tag(z.dtype), rows, inner, so,
                     si, vocab, tgt.data_ptr(), temperature, logp.data_ptr(),
                     entropy.data_ptr() if with_entropy else None, state.data_ptr(),
                     state.data_ptr() + 4 * at, kernels=2 if size > at else 1,
                     work=(rows * (vocab * z.element_size() + 20), 0))
    return logp, entropy, state


@_register("token_logprobs_bwd(Tensor logits, Tensor target, Tensor state, Tensor? entropy, "
           "Tensor? g_logp, Tensor? g_entropy, float temperature) -> Tensor",
           lambda logits, *_: logits.new_empty(logits.shape))
def token_logprobs_bwd(logits, target, state, entropy, g_logp, g_entropy, temperature):
    shape, at = logits.shape[:-1], logits.get_device()
    _need(target.get_device() == at and target.dtype == torch.int64 and target.shape == shape
          and state.get_device() == at and state.dtype == F32 and state.is_contiguous()
          and state.numel() >= 2 * target.numel() and _fits(entropy, at, F32, shape)
          and all(g is None or (g.get_device() == at and g.dtype == F32 and g.shape == shape)
                  for g in (g_logp, g_entropy)),
          "token_logprobs_bwd", "target, state, entropy and gradients as the forward has them")
    z, rows, inner, so, si = row_layout(logits)
    vocab, dev = logits.shape[-1], logits.device
    out = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
    if rows:
        tgt = target.contiguous()
        gl = g_logp.contiguous() if g_logp is not None else None
        ge = g_entropy.contiguous() if g_entropy is not None else None
        _lib.call_on(dev, "qb_token_logprobs_bwd", z.data_ptr(), _lib.tag(z.dtype), rows, inner,
                     so, si, vocab, tgt.data_ptr(), temperature, state.data_ptr(),
                     _lib.ptr(entropy), _lib.ptr(gl), _lib.ptr(ge), out.data_ptr(),
                     work=(rows * (2 * vocab * z.element_size() + 28), 0))
    return out


# ------------------------------------------------------------------------------------------
# preference loss


class _Preference(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logp, mask, *args):
        loss, state = preference.below(logp, mask, *args)
        ctx.save_for_backward(mask, state)
        ctx.shape, ctx.dtype, ctx.args = logp.shape, logp.dtype, len(args)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(state)
        return loss, state

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _g_state):
        mask, state = ctx.saved_tensors
        none = (None,) * (ctx.args + 1)
        if g is None:
            return None, *none
        return preference_bwd(state, mask, g, *ctx.shape, ctx.dtype), *none


def preference_state(n, cols):
    """Floats of the second output (rewards [n], coefficients [n], workspace), the workspace's
    offset."""
    at = _up4(2 * n)
    return at + 4 * n * ((cols + 2047) // 2048), at


def _preference_fake(logp, *_):
    return logp.new_empty((), dtype=F32), logp.new_empty((preference_state(*logp.shape)[0],),
                                                         dtype=F32)


@_register("preference(Tensor logp, Tensor? mask, Tensor? ref, Tensor? ref_row, "
           "Tensor? denominator, float beta, float label_smoothing, float margin, "
           "float divide_by, int loss_type, bool length_normalized) -> (Tensor, Tensor)",
           _preference_fake, _Preference)
def preference(logp, mask, ref, ref_row, denominator, beta, label_smoothing, margin, divide_by,
               loss_type, length_normalized):
    n, cols = logp.shape
    dev = logp.device
    here = logp.get_device()
    _need(n % 2 == 0 and logp.is_contiguous() and _fits(ref, here, logp.dtype, logp.shape)
          and (ref_row is None or ref_row.dtype in (F32, F64)
               and _fits(ref_row, here, ref_row.dtype, (n,)))
          and _fits(denominator, here, F64, ())
          and _mask_fits(mask, here, logp.shape), "preference",
          "pairs of rows, contiguous tensors on one device: ref in logp's dtype, ref_row fp32 or "
          "fp64, bool or byte mask, double denominator")
    loss = torch.empty((), dtype=F32, device=dev)
    size, at = preference_state(n, cols)
    state = torch.empty(size, dtype=F32, device=dev)
    base = state.data_ptr()
    cfg = PreferenceConfig(beta, label_smoothing, margin, divide_by, loss_type,
                           length_normalized)
    e = logp.element_size()
    _lib.call_on(dev, "qb_preference_fwd", logp.data_ptr(), _lib.ptr(ref), _lib.tag(logp.dtype),
                 _lib.ptr(mask), _lib.ptr(ref_row),
                 int(ref_row is not None and ref_row.dtype == F64), n // 2, cols,
                 ctypes.addressof(cfg),
                 _lib.ptr(denominator), loss.data_ptr(), base, base + 4 * n, base + 4 * at,
                 kernels=2,
                 work=(n * cols * (e * (1 if ref is None else 2) + (mask is not None)), 0))
    return loss, state


@_register("preference_bwd(Tensor state, Tensor? mask, Tensor g, SymInt n, SymInt cols, "
           "ScalarType dtype) -> Tensor",
           lambda state, mask, g, n, cols, dtype: state.new_empty((n, cols), dtype=dtype))
def preference_bwd(state, mask, g, n, cols, dtype):
    here = state.get_device()
    _need(n % 2 == 0 and state.dtype == F32 and state.is_contiguous() and state.numel() >= 2 * n
          and _fits(g, here, F32, ()) and _mask_fits(mask, here, (n, cols)),
          "preference_bwd", "pairs of rows; state, mask and gradient as the forward has them")
    out = torch.empty((n, cols), dtype=dtype, device=state.device)
    _lib.call_on(state.device, "qb_preference_bwd", _lib.ptr(mask), state.data_ptr() + 4 * n,
                 g.data_ptr(), n // 2, cols, out.data_ptr(), _lib.tag(dtype),
                 work=(n * cols * (out.element_size() + (mask is not None)), 0))
    return out


# ------------------------------------------------------------------------------------------
# clipped policy loss


class _Policy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logp, *args):
        loss, state, unit = policy.below(logp, *args)
        ctx.save_for_backward(state, unit)
        ctx.dtype, ctx.args, ctx.sequence, ctx.with_grad = logp.dtype, len(args), *args[-2:]
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(state, unit)
        return loss, state, unit

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _g_state, _g_unit):
        state, unit = ctx.saved_tensors
        none = (None,) * ctx.args
        if g is None:
            return None, *none
        if not ctx.with_grad:
            raise RuntimeError("qlora_b200::policy: backward through a call made without the "
                               "gradient (with_grad=False)")
        return policy_bwd(unit, state, g, ctx.sequence, ctx.dtype), *none


def policy_state(n, cols, sequence):
    """Floats of the second output (statistics [4], weights [n] or one, workspace), the workspace's
    offset."""
    at = _up4(4 + (n if sequence else 1))
    return at + 8 * n * ((cols + 2047) // 2048), at


def _policy_fake(logp, old_logp, advantages, mask, ref, denominator, clip_low, clip_high, delta,
                 kl_coef, divide_by, sequence, with_grad):
    n, cols = logp.shape
    return (logp.new_empty((), dtype=F32),
            logp.new_empty((policy_state(n, cols, sequence)[0],), dtype=F32),
            logp.new_empty((n if with_grad else 0, cols), dtype=F32))


@_register("policy(Tensor logp, Tensor? old_logp, Tensor advantages, Tensor? mask, Tensor? ref, "
           "Tensor? denominator, float clip_low, float clip_high, float delta, float kl_coef, "
           "float divide_by, bool sequence, bool with_grad) -> (Tensor, Tensor, Tensor)",
           _policy_fake, _Policy)
def policy(logp, old_logp, advantages, mask, ref, denominator, clip_low, clip_high, delta,
           kl_coef, divide_by, sequence, with_grad):
    n, cols = logp.shape
    dev = logp.device
    here = logp.get_device()
    _need(logp.is_contiguous() and _fits(old_logp, here, logp.dtype, logp.shape)
          and _fits(ref, here, logp.dtype, logp.shape) and _mask_fits(mask, here, logp.shape)
          and _fits(denominator, here, F64, ())
          and advantages.get_device() == here and advantages.dtype == F32
          and advantages.shape in ((n,), (n, cols)), "policy",
          "contiguous tensors on one device: old_logp and ref in logp's dtype, fp32 advantages, "
          "bool or byte mask, double denominator")
    loss = torch.empty((), dtype=F32, device=dev)
    size, at = policy_state(n, cols, sequence)
    state = torch.empty(size, dtype=F32, device=dev)
    base = state.data_ptr()
    unit = torch.empty((n if with_grad else 0, cols), dtype=F32, device=dev)
    cfg = PolicyConfig(clip_low, clip_high, delta, kl_coef, divide_by, sequence, 0)
    per_token = advantages.dim() == 2
    arrays = 1 + (old_logp is not None) + (ref is not None)
    _lib.call_on(dev, "qb_policy_fwd", logp.data_ptr(), _lib.ptr(old_logp), _lib.ptr(ref),
                 _lib.tag(logp.dtype), advantages.data_ptr(), advantages.stride(0),
                 advantages.stride(1) if per_token else 0, _lib.ptr(mask), n, cols,
                 ctypes.addressof(cfg), _lib.ptr(denominator), loss.data_ptr(), base, base + 16,
                 unit.data_ptr() if with_grad else None, base + 4 * at, kernels=2,
                 work=(n * cols * (arrays * logp.element_size() + 4 * per_token + 4 * with_grad
                                   + (mask is not None)), 0))
    return loss, state, unit


@_register("policy_bwd(Tensor unit, Tensor state, Tensor g, bool sequence, ScalarType dtype) "
           "-> Tensor",
           lambda unit, state, g, sequence, dtype: unit.new_empty(unit.shape, dtype=dtype))
def policy_bwd(unit, state, g, sequence, dtype):
    n, cols = unit.shape
    here = unit.get_device()
    _need(unit.dtype == F32 and unit.is_contiguous() and _fits(g, here, F32, ())
          and state.get_device() == here and state.dtype == F32 and state.is_contiguous()
          and state.numel() >= 4 + (n if sequence else 1), "policy_bwd",
          "unit gradient, state and gradient as the forward has them")
    out = torch.empty((n, cols), dtype=dtype, device=unit.device)
    _lib.call_on(unit.device, "qb_policy_bwd", unit.data_ptr(), state.data_ptr() + 16,
                 int(sequence), g.data_ptr(), n, cols, out.data_ptr(), _lib.tag(dtype),
                 work=(n * cols * (4 + out.element_size()), 0))
    return out


def ops():
    """Every op of this module (for checks such as torch.library.opcheck)."""
    return {name: getattr(torch.ops.qlora_b200, name) for name in (
        "token_logprobs", "token_logprobs_bwd", "preference", "preference_bwd", "policy",
        "policy_bwd")}


# ------------------------------------------------------------------------------------------
# argument checks the objectives share


def constant(what, name, t, logp):
    """`t` as a constant of an objective over `logp`: on its device, no part of a graph."""
    if t.device != logp.device:
        raise ValueError(f"{what}: {name} is on {t.device}, logp on {logp.device}")
    if t.requires_grad:
        raise ValueError(f"{what}: {name} is a constant of the objective (no gradient flows into "
                         "it); pass it detached")
    return t


def mask_bytes(what, mask, logp):
    """The mask as contiguous bytes (nonzero: the token counts), or None."""
    if mask is None:
        return None
    if mask.shape != logp.shape or mask.device != logp.device:
        raise ValueError(f"{what}: mask {tuple(mask.shape)} on {mask.device} for logp "
                         f"{tuple(logp.shape)} on {logp.device}")
    if mask.dtype not in (torch.bool, torch.uint8):
        mask = mask != 0
    return mask.contiguous()


def divisor(what, denominator, device):
    """(device double or None, number or 0.0) of a denominator given as a tensor, a number or
    None. A tensor is not read on the host."""
    if denominator is None:
        return None, 0.0
    if torch.is_tensor(denominator):
        if denominator.numel() != 1:
            raise ValueError(f"{what}: the denominator is one number")
        if denominator.requires_grad:
            raise ValueError(f"{what}: the denominator is a constant of the objective (no gradient "
                             "flows into it); pass it detached")
        return denominator.reshape(()).to(device=device, dtype=torch.float64), 0.0
    value = float(denominator)
    if not 0.0 < value < float("inf"):
        raise ValueError(f"{what}: denominator {denominator} is not positive")
    return None, value


def logp_matrix(what, logp):
    """logp as the objectives read it: a CUDA [rows, tokens] matrix of a kernel dtype."""
    _lib.require_cuda(logp, what=what)
    if logp.dim() != 2 or logp.shape[0] == 0 or logp.shape[1] == 0:
        raise ValueError(f"{what}: logp is [rows, tokens], got {tuple(logp.shape)}")
    _lib.tag(logp.dtype)
    return logp
