"""The global gradient norm and clipping (grad_norm.py) against 64-bit sums.

The sums are 64-bit (relative errors of about n 2^-53, nothing beside fp32's), so the returned
norm is off by its rounding to fp32: u = 2^-24 relative, and u more for the 64-bit reference's own
sums. A clipped gradient is g * coef with coef rounded to fp32 (u), the product rounded in fp32
(u) and, for 16-bit types, rounded again (half a step of theirs)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
ORDERS = [2.0, 1.0, math.inf]


def params_of(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty(g.shape, dtype=g.dtype, device=g.device))
        p.grad = g
        out.append(p)
    return out


def norm64(grads, order):
    flat = torch.cat([g.detach().double().reshape(-1) for g in grads])
    return float(torch.linalg.vector_norm(flat, order)) if flat.numel() else 0.0


def check(grads, order=2.0, share=0.3):
    from hackathon_b200.grad_norm import clip_grad_norm_, grad_norm
    before = [g.detach().clone() for g in grads]
    want = norm64(before, order)
    norm = grad_norm(grads, order)
    assert norm.dtype == torch.float32 and norm.shape == ()
    assert abs(float(norm) - want) <= 2 * U * want
    for limit in (share * want, 2 * want + 1.0):
        for g, b in zip(grads, before):
            g.copy_(b)
        got = clip_grad_norm_(params_of(grads), limit, order)
        assert float(got) == float(norm)
        coef = min(1.0, limit / (want + 1e-6))
        for g, b in zip(grads, before):
            if coef == 1.0:
                assert torch.equal(g, b)
                continue
            exact = b.double() * coef
            tol = exact.abs() * (3 * U + HALF[g.dtype]) + torch.finfo(g.dtype).smallest_normal
            assert bool(((g.double() - exact).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("sizes", [(1,), (7,), (8191, 8192, 8193), (3, 0, 70001, 1),
                                   (16, 896, 14336, 131072)], ids=str)
def test_norm_and_clipping(cuda, sizes, order, dtype):
    g = torch.Generator(device=cuda).manual_seed(sum(sizes))
    check([torch.randn(n, device=cuda, generator=g).to(dtype) for n in sizes], order)


def test_types_side_by_side_and_odd_addresses(cuda):
    """Three types in one call, each tensor starting at an odd place of its buffer, neighbours
    untouched."""
    g = torch.Generator(device=cuda).manual_seed(2)
    from hackathon_b200.grad_norm import clip_grad_norm_
    for n in (1, 5, 8192, 8193, 30011):
        bufs = [torch.randn(n + 24, device=cuda, generator=g).to(d)
                for d in (torch.float32, torch.bfloat16, torch.float16)]
        for off in (1, 2, 3, 5, 7):
            copies = [b.clone() for b in bufs]
            check([b[off: off + n] for b in copies])
            clip_grad_norm_(params_of([b[off: off + n] for b in copies]), 1e-3)
            for b, c in zip(bufs, copies):
                assert torch.equal(b[:off], c[:off]) and torch.equal(b[off + n:], c[off + n:])


@pytest.mark.parametrize("n", [95, 96, 97, 1599, 1600, 1601, 3301])
def test_many_tensors(cuda, n):
    """Counts around the sizes of the launch tables."""
    g = torch.Generator(device=cuda).manual_seed(n)
    flat = torch.randn(sum(i % 41 for i in range(n)), device=cuda, generator=g)
    at, grads = 0, []
    for i in range(n):
        grads.append(flat[at: at + i % 41])
        at += i % 41
    check(grads)


def test_large_tensor_past_32_bit_offsets(cuda):
    from hackathon_b200.grad_norm import clip_grad_norm_
    n = (1 << 32) + 12345
    x = torch.zeros(n, dtype=torch.bfloat16, device=cuda)
    at = [0, 1 << 31, (1 << 32) - 1, 1 << 32, n - 1]
    x[at] = torch.tensor([3.0, 4.0, 12.0, 84.0, 132.0], dtype=torch.bfloat16, device=cuda)
    want = math.sqrt(3 ** 2 + 4 ** 2 + 12 ** 2 + 84 ** 2 + 132 ** 2)
    (p,) = params_of([x])
    assert abs(float(clip_grad_norm_(p, want / 2)) - want) <= 2 * U * want
    assert x[at].tolist() == [1.5, 2.0, 6.0, 42.0, 66.0]


def test_layouts(cuda):
    """Transposed gradients are one run of memory; gaps go through a copy; expanded ones have a
    norm but cannot be scaled in place."""
    from hackathon_b200.grad_norm import clip_grad_norm_, grad_norm
    g = torch.Generator(device=cuda).manual_seed(4)
    x = torch.randn(40, 30, device=cuda, generator=g)
    check([x.t(), torch.randn(5, 6, 7, device=cuda, generator=g).permute(2, 0, 1)])
    buf = x.clone()
    check([x[:, ::3], torch.randn(3, device=cuda, generator=g)])
    keep = torch.ones(30, dtype=torch.bool, device=cuda)
    keep[::3] = False
    assert torch.equal(x[:, keep], buf[:, keep])
    e = torch.randn(3, 1, device=cuda, generator=g).expand(3, 4)
    assert abs(float(grad_norm(e)) - norm64([e], 2.0)) <= 2 * U * norm64([e], 2.0)
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm_(params_of([e]), 1.0)


def test_shared_gradients_are_refused(cuda):
    from hackathon_b200.grad_norm import clip_grad_norm_
    x = torch.ones(100, device=cuda)
    for grads in ([x, x], [x[:60], x[50:]], [x[50:], x[:51]]):
        with pytest.raises(RuntimeError, match="share memory"):
            clip_grad_norm_(params_of(grads), 1.0)
    assert torch.equal(x, torch.ones_like(x))
    clip_grad_norm_(params_of([x[50:], x[:50]]), 1.0)       # neighbours are fine, in any order


def test_values_at_the_ends_of_the_range(cuda):
    """Squares that overflow or vanish in fp32."""
    for v in (1e30, 3e38, 1e-30, 1e-42):
        x = torch.full((9000,), v, device=cuda)
        want = float(x[0].double()) * math.sqrt(9000)
        from hackathon_b200.grad_norm import grad_norm
        got = float(grad_norm(x))
        if want > 3.4028234e38:
            assert got == math.inf
        else:
            assert abs(got - want) <= 2 * U * want + 2.0 ** -149


@pytest.mark.parametrize("order", ORDERS)
def test_infinite_and_nan_gradients(cuda, order):
    from hackathon_b200.grad_norm import clip_grad_norm_, grad_norm
    for bad in (math.inf, -math.inf, math.nan):
        for at in (0, 8191, 20000):
            x = torch.ones(20001, device=cuda)
            y = torch.ones(10, device=cuda)
            x[at] = bad
            norm = float(grad_norm([x, y], order))
            assert math.isnan(norm) if math.isnan(bad) else norm == math.inf
            with pytest.raises(RuntimeError, match="norm is"):
                clip_grad_norm_(params_of([x, y]), 1.0, order, error_if_nonfinite=True)
            assert torch.equal(y, torch.ones_like(y))
            clip_grad_norm_(params_of([x, y]), 1.0, order)
            # as the formula: a NaN spreads everywhere, an infinity leaves zeros and a NaN
            assert torch.isnan(x[at])
            assert torch.isnan(y).all() if math.isnan(bad) else not y.any()


def test_no_gradients(cuda):
    from hackathon_b200.grad_norm import clip_grad_norm_, grad_norm
    p = torch.nn.Parameter(torch.ones(3, device=cuda))
    assert float(clip_grad_norm_([p], 1.0)) == 0.0
    p.grad = torch.zeros_like(p)
    assert float(clip_grad_norm_([p], 1.0)) == 0.0 and not p.grad.any()
    assert float(clip_grad_norm_([p], 0.0)) == 0.0
    empty = torch.empty(0, device=cuda)
    assert float(grad_norm([empty])) == 0.0 and grad_norm([empty]).is_cuda
    p.grad = torch.ones_like(p)
    assert abs(float(clip_grad_norm_([p], 0.0)) - math.sqrt(3)) < 1e-6 and not p.grad.any()


def test_same_bits_stream_graph_and_version(cuda):
    from hackathon_b200.grad_norm import clip_grad_norm_
    g = torch.Generator(device=cuda).manual_seed(8)
    src = [torch.randn(n, device=cuda, generator=g) for n in (14336, 3, 100003, 77)]
    work = [s.clone() for s in src]
    ps = params_of(work)

    def run():
        for w, s in zip(work, src):
            w.copy_(s)
        return clip_grad_norm_(ps, 0.5)

    version = work[0]._version
    norm = run()
    assert work[0]._version == version + 2
    first = [w.clone() for w in work]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, norm) and all(map(torch.equal, work, first))
    # two captured graphs, replayed in turn: each has its own table and workspace
    graphs = []
    for k in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    src[0].mul_(2.0)
    for graph, out in graphs * 2:
        for w in work:
            w.zero_()
        graph.replay()
        assert abs(float(out) - norm64(src, 2.0)) <= 2 * U * norm64(src, 2.0)
        assert abs(norm64(work, 2.0) - 0.5) < 1e-5


def test_timer_counts_the_bytes_that_moved(cuda):
    """A kernel timer's bytes: one pass for a norm and for a clipping within the limit, the norm's
    read and the scaling's read and write where it scales."""
    from hackathon_b200 import _lib
    from hackathon_b200.grad_norm import clip_grad_norm_, grad_norm
    grads = [torch.ones(300, device=cuda), torch.ones(100, device=cuda, dtype=torch.bfloat16)]
    size, ps = 300 * 4 + 100 * 2, params_of(grads)
    for limit, passes in ((1e3, 1), (1.0, 3), (math.inf, 1), (0.0, 3)):
        for g in grads:
            g.fill_(1.0)
        with _lib.KernelTimer() as timer:
            clip_grad_norm_(ps, limit).zero_()          # the caller's to write to
        assert timer.summary()["qb_grad_clip"]["bytes"] == passes * size
    grads[0][7] = math.nan
    with _lib.KernelTimer() as timer:
        grad_norm(grads)
        clip_grad_norm_(ps, 1e3)
    both = timer.summary()
    assert both["qb_grad_norm"]["bytes"] == size and both["qb_grad_clip"]["bytes"] == 3 * size
