"""The post-training operators without a GPU: shapes through their fake implementations, the
C-ABI's layouts and refusals (made before any CUDA call), and the argument checks of the
functions users call."""

import ctypes
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import hackathon_b200.objective_ops as oo
from hackathon_b200 import _lib
from hackathon_b200.grad_norm import clip_grad_norm_, grad_norm
from hackathon_b200.logprobs import linear_token_logprobs, token_logprobs
from hackathon_b200.policy import policy_loss
from hackathon_b200.preference import preference_loss

F32, BF, I64 = torch.float32, torch.bfloat16, torch.int64


def test_ops_are_registered_beside_the_others():
    import hackathon_b200.ops as qops
    assert set(oo.ops()) == {"token_logprobs", "token_logprobs_bwd", "preference",
                             "preference_bwd", "policy", "policy_bwd"}
    assert not set(oo.ops()) & set(qops.ops())


def test_fake_implementations_give_the_output_shapes():
    with FakeTensorMode():
        def e(*s, dtype=F32):
            return torch.empty(s, dtype=dtype, device="cuda")
        lp, en = token_logprobs(e(2, 5, 30, dtype=BF), e(2, 5, dtype=I64), 0.7, True)
        assert lp.shape == en.shape == (2, 5) and lp.dtype == en.dtype == F32
        assert token_logprobs(e(30), e(dtype=I64)).shape == ()
        loss, step = preference_loss(e(6, 9, dtype=BF), e(6, 9, dtype=torch.bool), e(6, 9))
        assert loss.shape == () and loss.dtype == F32
        assert step.chosen_rewards.shape == step.rejected_rewards.shape == (3,)
        assert step.margins.shape == (3,) and step.accuracy.shape == ()
        for reduction in ("token", "sequence"):
            loss, step = policy_loss(e(4, 7), e(4, 7), e(4), reduction=reduction)
            assert loss.shape == step.kl.shape == step.tokens.shape == ()


def test_gradients_have_the_inputs_shapes_on_meta_tensors():
    def e(*s, dtype=F32, grad=False):
        return torch.empty(*s, dtype=dtype, device="meta", requires_grad=grad)
    z = e(2, 5, 30, dtype=BF, grad=True)
    lp, en, _ = oo.token_logprobs(z, e(2, 5, dtype=I64), 1.0, True)
    (g,) = torch.autograd.grad((lp + en).sum(), z)
    assert g.shape == z.shape and g.dtype == BF
    for op, args in ((oo.preference, (None, None, None, None, 0.1, 0.0, 0.0, 0.0, 0, False)),
                     (oo.policy, (None, e(6), None, None, None, 0.2, 0.2, 0.0, 0.0, 0.0, True,
                                  True))):
        x = e(6, 9, dtype=torch.float16, grad=True)
        (g,) = torch.autograd.grad(op(x, *args)[0], x)
        assert g.shape == x.shape and g.dtype == x.dtype
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        x = e(6, 9, grad=True)
        loss = oo.preference(x, None, None, None, None, 0.1, 0.0, 0.0, 0.0, 0, False)[0]
        (g,) = torch.autograd.grad(loss, x, create_graph=True)
        torch.autograd.grad(g.sum(), x)


@pytest.mark.parametrize("n,cols", [(2, 1), (6, 2048), (6, 2049), (10, 70001), (2, 151936),
                                    (300, 50001), (592, 8193), (1184, 40000), (5000, 152064)])
def test_state_layout_matches_the_library(n, cols):
    """The buffers the ops allocate hold what the library says its workspace needs, at an aligned
    offset, and the fake implementations give their sizes."""
    lib = _lib.load()
    assert lib.qb_preference_config_size() == ctypes.sizeof(oo.PreferenceConfig)
    assert lib.qb_policy_config_size() == ctypes.sizeof(oo.PolicyConfig)
    meta = torch.empty(n, cols, device="meta")
    target = torch.empty(n, device="meta", dtype=I64)
    for dtype, tag in ((F32, 0), (torch.float16, 1), (BF, 2)):
        size, at = oo.logprobs_state(n, cols, dtype.itemsize)
        assert at >= 2 * n and at % 4 == 0
        assert 4 * (size - at) >= lib.qb_token_logprobs_workspace(n, cols, tag)
        assert (size > at) >= (lib.qb_token_logprobs_workspace(n, cols, tag) > 0)
        assert oo._token_logprobs_fake(meta.to(dtype), target, 1.0, True)[2].shape == (size,)
    size, at = oo.preference_state(n, cols)
    assert at >= 2 * n and at % 4 == 0
    assert 4 * (size - at) == lib.qb_preference_workspace(n // 2, cols)
    assert oo._preference_fake(meta)[1].shape == (size,)
    for sequence in (False, True):
        size, at = oo.policy_state(n, cols, sequence)
        assert at >= 4 + (n if sequence else 1) and at % 4 == 0
        assert 4 * (size - at) == lib.qb_policy_workspace(n, cols)
        got = oo._policy_fake(meta, *(None,) * 10, sequence, True)
        assert got[1].shape == (size,) and got[2].shape == (n, cols)


def test_row_layout_reads_views_in_place():
    x = torch.empty(3, 5, 8)

    def starts(t):
        z, rows, inner, so, si = oo.row_layout(t)
        return z, [z.storage_offset() + (r // inner) * so + (r % inner) * si
                   for r in range(rows)]

    z, at = starts(x)
    assert z is x and at == [8 * r for r in range(15)]
    z, at = starts(x[:, :-1])
    assert z.data_ptr() == x.data_ptr()
    assert at == [b * 40 + s * 8 for b in range(3) for s in range(4)]
    z, at = starts(x[:, 1:, :7])
    assert at == [b * 40 + (s + 1) * 8 for b in range(3) for s in range(4)]
    z, at = starts(x[:, 0])
    assert z.data_ptr() == x.data_ptr() and at == [0, 40, 80]
    z, at = starts(x[0, 0].expand(4, 8))
    assert at == [0, 0, 0, 0]
    z, at = starts(torch.empty(8))
    assert len(at) == 1
    z, at = starts(torch.empty(2, 3, 4, 8))
    assert at == [8 * r for r in range(24)]
    z, at = starts(torch.empty(2, 8, 3).transpose(1, 2))       # the vocabulary is not contiguous
    assert z.is_contiguous() and len(at) == 6
    assert starts(torch.empty(0, 5, 8))[1] == [] and starts(torch.empty(2, 0, 8))[1] == []


def test_c_entries_refuse_before_any_launch():
    fake = 1 << 20
    keep = []

    def lp(rows=4, inner=1, vocab=10, t=1.0, dtype=0, logits=fake, out=fake):
        return ("qb_token_logprobs", logits, dtype, rows, inner, vocab, 0, vocab, fake, t, out,
                None, fake, fake, None)

    cases = [(lp(vocab=0), "bad shape"), (lp(rows=-1), "bad shape"), (lp(inner=0), "bad shape"),
             (lp(inner=3), "bad shape"), (lp(vocab=1 << 30), "bad shape"),
             (lp(t=0.0), "temperature"), (lp(t=math.nan), "temperature"),
             (lp(t=math.inf), "temperature"), (lp(logits=None), "null"), (lp(out=None), "null"),
             (lp(dtype=7), "unsupported dtype"),
             (lp(rows=(1 << 31)), "too many rows")]
    cases += [(("qb_token_logprobs_bwd", fake, 0, 4, 1, 10, 0, 10, fake, 1.0, fake, e, fake, ge,
                out, None), "null") for e, ge, out in ((None, fake, fake), (fake, fake, None))]
    pref = oo.PreferenceConfig(0.1, 0.0, 0.0, 0.0, 0, 0)

    def pr(cfg=pref, pairs=2, cols=8, ref=None, row=None, logp=fake, **kw):
        keep.append(cfg)               # the call reads it at its address
        at = ctypes.addressof(cfg) if cfg is not None else None
        return ("qb_preference_fwd", logp, ref, 0, None, row, 0, pairs, cols, at, None, fake, fake,
                fake, fake, None)

    cases += [(pr(pairs=0), "bad shape"), (pr(cols=0), "bad shape"), (pr(logp=None), "null"),
              (pr(cfg=None), "null"), (pr(pairs=1 << 29, cols=1 << 20), "too large"),
              (pr(ref=fake, row=fake), "two references")]
    for bad in (oo.PreferenceConfig(0.0, 0, 0, 0, 0, 0), oo.PreferenceConfig(0.1, 0.5, 0, 0, 0, 0),
                oo.PreferenceConfig(0.1, 0, math.nan, 0, 0, 0),
                oo.PreferenceConfig(0.1, 0, 0, 0, 3, 0)):
        cases.append((pr(cfg=bad), "bad loss type"))
    cases.append((("qb_preference_bwd", None, None, fake, 2, 8, fake, 0, None), "null"))

    def po(cfg, rows=2, cols=8, adv=fake):
        keep.append(cfg)
        return ("qb_policy_fwd", fake, fake, None, 0, adv, 1, 0, None, rows, cols,
                ctypes.addressof(cfg), None, fake, fake, fake, fake, fake, None)

    good = oo.PolicyConfig(0.2, 0.2, 0.0, 0.0, 0.0, 0, 0)
    cases += [(po(good, rows=0), "bad shape"), (po(good, adv=None), "null"),
              (po(good, rows=1 << 31), "too large")]
    for bad in (oo.PolicyConfig(1.1, 0.2, 0, 0, 0, 0, 0), oo.PolicyConfig(0.2, -0.1, 0, 0, 0, 0, 0),
                oo.PolicyConfig(0.2, 0.2, 1.1, 0, 0, 0, 0),
                oo.PolicyConfig(0.2, 0.2, 0, math.nan, 0, 0, 0),
                oo.PolicyConfig(0.2, 0.2, 0, 0, 0, 2, 0)):
        cases.append((po(bad), "bad clip range"))
    cases.append((("qb_policy_bwd", fake, None, 0, fake, 2, 8, fake, 0, None), "null"))

    def table(ptrs, sizes, tags):
        n = len(ptrs)
        return ((ctypes.c_uint64 * n)(*ptrs), (ctypes.c_int64 * n)(*sizes), bytes(tags), n)

    def clip(ptrs, sizes, tags, order=2, limit=1.0):
        keep.append(ctypes.c_double(limit))
        return ("qb_grad_clip", *table(ptrs, sizes, tags), order, ctypes.addressof(keep[-1]),
                fake, 1 << 20, fake, None)

    cases += [(("qb_grad_norm", None, None, None, 1, 2, fake, 99, fake, None), "null"),
              (("qb_grad_norm", *table([fake], [4], [0]), 2, fake, 0, fake, None), "too small"),
              (("qb_grad_norm", *table([fake], [4], [0]), 3, fake, 99, fake, None), "order"),
              (("qb_grad_norm", *table([fake], [4], [5]), 2, fake, 99, fake, None), "dtype"),
              (("qb_grad_norm", *table([fake + 2], [4], [0]), 2, fake, 99, fake, None),
               "misaligned"),
              (("qb_grad_norm", *table([0], [4], [0]), 2, fake, 99, fake, None), "null or"),
              (("qb_grad_norm", *table([fake], [-4], [0]), 2, fake, 99, fake, None), "bad size"),
              (clip([fake, fake], [4, 4], [0, 0]), "share memory"),
              (clip([fake + 64, fake], [4, 17], [0, 0]), "share memory"),
              (clip([fake], [4], [0], limit=-1.0), "max_norm"),
              (clip([fake], [4], [0], limit=math.nan), "max_norm")]
    for args, match in cases:
        with pytest.raises(RuntimeError, match=match):
            _lib.call(*args)
    # nothing to do is no error
    assert _lib.load().qb_token_logprobs(None, 0, 0, 1, 10, 0, 10, None, 1.0, None, None, None,
                                         None, None) == 0
    assert _lib.load().qb_preference_workspace(0, 5) == 0
    assert _lib.load().qb_policy_workspace(4, 0) == 0


def _fake_cuda(fn):
    with FakeTensorMode():
        fn(lambda *s, dtype=F32, **k: torch.empty(*s, dtype=dtype, device="cuda", **k))


def test_token_logprobs_refusals():
    def run(e):
        t = e(2, 5, dtype=I64)
        with pytest.raises(RuntimeError, match="CUDA"):
            token_logprobs(torch.empty(2, 5, 30, device="cpu"), t)
        with pytest.raises(TypeError, match="dtype"):
            token_logprobs(e(2, 5, 30, dtype=torch.float64), t)
        with pytest.raises(ValueError, match="target"):
            token_logprobs(e(2, 4, 30), t)
        with pytest.raises(ValueError, match="target"):
            token_logprobs(e(2, 5, 0), t)
        with pytest.raises(TypeError, match="token numbers"):
            token_logprobs(e(2, 5, 30), e(2, 5))
        for bad in (0.0, -1.0, math.nan, math.inf):
            with pytest.raises(ValueError, match="temperature"):
                token_logprobs(e(2, 5, 30), t, bad)
        for h, w, target in ((e(2, 5, 8), e(30, 8), t[:, :4]), (e(2, 5, 8), e(30, 9), t),
                             (e(2, 5, 8), e(8), t), (e(2, 5, 8), e(30, 8), t.reshape(10))):
            with pytest.raises(ValueError, match="linear_token_logprobs"):
                linear_token_logprobs(h, w, target)
    _fake_cuda(run)
    with pytest.raises(RuntimeError, match="CUDA"):
        linear_token_logprobs(torch.ones(2, 8), torch.ones(10, 8), torch.ones(2, dtype=I64))


def test_preference_refusals():
    def run(e):
        x = e(4, 6)
        with pytest.raises(RuntimeError, match="CUDA"):
            preference_loss(torch.empty(4, 6, device="cpu"))
        for bad, match in ((dict(beta=0.0), "beta"), (dict(beta=math.nan), "beta"),
                           (dict(loss_type="kto"), "loss_type"),
                           (dict(label_smoothing=0.5), "smoothing"),
                           (dict(label_smoothing=0.1, loss_type="hinge"), "smoothing"),
                           (dict(margin=1.0, loss_type="ipo"), "margin"),
                           (dict(margin=math.inf), "margin"),
                           (dict(denominator=0), "denominator"),
                           (dict(denominator=e(2)), "denominator"),
                           (dict(mask=e(4, 5)), "mask"), (dict(ref_logp=e(4, 5)), "ref_logp"),
                           (dict(ref_logp=e(2)), "ref_logp"),
                           (dict(ref_logp=e(4, 6, requires_grad=True)), "detached")):
            with pytest.raises(ValueError, match=match):
                preference_loss(x, **bad)
        for shape in ((3, 6), (4,), (0, 6), (4, 0)):
            with pytest.raises(ValueError):
                preference_loss(e(*shape))
        with pytest.raises(TypeError):
            preference_loss(e(4, 6, dtype=torch.float64))
        with pytest.raises(TypeError):
            preference_loss(x, ref_logp=e(4, 6, dtype=torch.float64))
    _fake_cuda(run)


def test_policy_refusals():
    def run(e):
        x, a = e(4, 6), e(4)
        with pytest.raises(RuntimeError, match="CUDA"):
            policy_loss(torch.empty(4, 6, device="cpu"), x, a)
        for bad, match in ((dict(clip_low=1.5), "clip"), (dict(clip_low=-0.1), "clip"),
                           (dict(clip_high=-0.1), "clip"), (dict(clip_high=math.inf), "clip"),
                           (dict(delta=1.1), "delta"), (dict(delta=math.nan), "delta"),
                           (dict(kl_coef=0.1), "ref_logp"),
                           (dict(kl_coef=math.nan, ref_logp=x), "kl_coef"),
                           (dict(reduction="mean"), "reduction"),
                           (dict(denominator=-3), "denominator"), (dict(mask=e(4)), "mask"),
                           (dict(ref_logp=e(4, 5)), "ref_logp"),
                           (dict(ref_logp=e(4, 6, requires_grad=True)), "detached")):
            with pytest.raises(ValueError, match=match):
                policy_loss(x, x, a, **bad)
        with pytest.raises(ValueError, match="old_logp"):
            policy_loss(x, e(4, 5), a)
        with pytest.raises(ValueError, match="advantages"):
            policy_loss(x, x, e(6))
        with pytest.raises(ValueError, match="advantages"):
            policy_loss(x, x, e(4, 1))
        with pytest.raises(ValueError, match="detached"):
            policy_loss(x, x, e(4, requires_grad=True))
    _fake_cuda(run)


def test_grad_norm_refusals():
    p = torch.nn.Parameter(torch.ones(3))
    assert float(clip_grad_norm_([p], 1.0)) == 0.0 and float(grad_norm([])) == 0.0
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="CUDA"):
        clip_grad_norm_(p, 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        grad_norm([p.grad])
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm_(p, bad)
    for bad in (0.0, 3.0, -math.inf, math.nan):
        with pytest.raises(ValueError, match="norm_type"):
            grad_norm(p.grad, bad)
    with pytest.raises(TypeError, match="dense"):
        grad_norm([torch.eye(3).to_sparse()])
    with pytest.raises(TypeError):
        grad_norm([p.grad, None])


def test_dense_layouts_are_recognised():
    from hackathon_b200.grad_norm import _fills_its_memory
    x = torch.empty(4, 6, 5)
    for t in (x, x.transpose(0, 2), x.permute(1, 2, 0), x[:1].transpose(0, 1), torch.empty(()),
              x.unsqueeze(1).expand(4, 1, 6, 5)):
        assert _fills_its_memory(t)
    for t in (x[:, :5], x[..., ::2], x[0, :1].expand(3, 5), x.unfold(2, 3, 1)):
        assert not _fills_its_memory(t)


def test_calls_run_on_the_tensors_device(monkeypatch):
    """A call for another device than the current one makes it the current one and passes its
    stream; a failing call raises the library's message either way."""
    entered, seen = [], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            entered.append(self.index)

        def __exit__(self, *exc):
            entered.append(None)

    class Lib:
        status = 0

        def qb_thing(self, *args):
            seen.append((args, list(entered)))
            return self.status

        def qb_last_error(self):
            return b"the reason"

    lib = Lib()
    monkeypatch.setattr(_lib, "_lib", lib)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    _lib.call_on(torch.device("cuda", 0), "qb_thing", 5)
    _lib.call_on(torch.device("cuda"), "qb_thing", 6)
    _lib.call_on(torch.device("cuda", 1), "qb_thing", 7)
    assert seen == [((5, 100), []), ((6, 100), []), ((7, 101), [1])] and entered == [1, None]
    lib.status = 1
    for index in (0, 1):
        with pytest.raises(RuntimeError, match="qb_thing failed .status 1.: the reason"):
            _lib.call_on(torch.device("cuda", index), "qb_thing")
    assert entered == [1, None, 1, None]


def test_second_launches_do_not_promise_read_only_memory():
    """A kernel that starts before the launch it follows has finished (await_previous) reads what
    that one writes: none of those pointers may be declared __restrict__, which would allow loads
    ahead of the wait and through the non-coherent path. Inputs older than both launches may."""
    import os
    import re
    root = os.path.join(os.path.dirname(_lib.__file__), "csrc")
    written = {"partials", "records"}
    found = 0
    for name in sorted(os.listdir(root)):
        if not name.endswith(".cu"):
            continue
        with open(os.path.join(root, name)) as f:
            text = f.read()
        for part in re.split(r"__global__", text)[1:]:
            head, _, body = part.partition("{")
            if "await_previous()" not in body.split("\n}\n")[0]:
                continue
            params = re.sub(r"\s+", " ", head[head.index("_kernel"):])
            names = {p: decl for decl in params.split(",")
                     for p in written if re.search(rf"\b{p}\b", decl)}
            assert names, f"{name}: {params}"
            for decl in names.values():
                assert "__restrict__" not in decl, f"{name}: {decl}"
            found += 1
    assert found == 5


def test_policy_second_border_of_zero_is_refused():
    """None is no second border; 0 is one below the others, not another word for None."""
    def run(e):
        for bad in (0, 0.0, -0.0):
            with pytest.raises(ValueError, match="delta"):
                policy_loss(e(4, 6), e(4, 6), e(4), delta=bad)
        policy_loss(e(4, 6), e(4, 6), e(4), delta=None)
    _fake_cuda(run)


def test_denominators_that_ask_for_a_gradient_are_refused():
    """As every other constant of an objective: its gradient would go nowhere."""
    def run(e):
        x, denom = e(4, 6), e((), requires_grad=True)
        with pytest.raises(ValueError, match="denominator.*detached"):
            policy_loss(x, x, e(4), denominator=denom)
        with pytest.raises(ValueError, match="denominator.*detached"):
            preference_loss(x, denominator=denom)
        policy_loss(x, x, e(4), denominator=denom.detach())
    _fake_cuda(run)


def test_linear_token_logprobs_targets_are_whole_numbers():
    """A target of another kind has no token: refused, as token_logprobs does, not cut off."""
    def run(e):
        for dtype in (F32, BF, torch.bool):
            with pytest.raises(TypeError, match="token numbers"):
                linear_token_logprobs(e(2, 5, 8), e(30, 8), e(2, 5, dtype=dtype))
        for dtype in (I64, torch.int32, torch.uint8):
            linear_token_logprobs(e(2, 5, 8), e(30, 8), e(2, 5, dtype=dtype))
    _fake_cuda(run)
