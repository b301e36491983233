"""The global gradient norm and clipping against 64-bit sums."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def norm_of(ts):
    return math.sqrt(sum(t.detach().double().square().sum().item() for t in ts))


# A thread adds up to 64 squares in float32, four sums of 16 one after the other, each square and sum rounded once: its sum
# of positive terms is off by less than 19 roundings of 2^-24 of it, the norm by half of that; all else is 64 bits, and the
# result is rounded once.
NORM = (19 / 2 + 1) * 2.0 ** -24


def check(got, ts):
    want = norm_of(ts)
    assert got.dtype == F32 and got.shape == ()
    assert abs(got.item() - want) <= NORM * want + 2.0 ** -149, (got.item(), want)


def check_scaled(out, g, norm, max_norm):
    """factor: a division and the rounding to float32; the product; and the rounding to out's type."""
    factor = min(1.0, max_norm / (norm + 1e-6))
    want = g.double() * factor
    half = torch.finfo(out.dtype).eps / 2
    allowed = want.abs() * (half + (NORM + 3 * 2.0 ** -24) * 1.01) + torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps
    assert ((out.double() - want).abs() <= allowed).all()


def make(g, shapes, dtypes, scale=1.0):
    return [(torch.randn(s, generator=g, device="cuda") * scale).to(dtypes[i % len(dtypes)]) for i, s in enumerate(shapes)]


SHAPES = [
    [(1,)], [(7,), (3, 5), ()], [(8192,)], [(8193,), (16383,), (1, 1)], [(512, 2048), (2048,), (512, 2048)], [(100003,)],
    [(0,), (5,), (0, 3)], [(97, 388), (388,)] * 40, [(3,)] * 2000, [(16384,)] * 65 + [(1,)],
]


@pytest.mark.parametrize("dtypes", [[F32], [BF16], [F16], [F16, F32, BF16]])
@pytest.mark.parametrize("shapes", SHAPES)
def test_norm_and_clipping(shapes, dtypes):
    from haste_b200 import gradients
    g = torch.Generator(device="cuda").manual_seed(len(shapes))
    ts = make(g, shapes, dtypes)
    norm = norm_of(ts)
    check(gradients.grad_norm(ts), ts)
    for bound in (norm / 2, norm * 2):
        outs = [torch.full(t.shape, 7.0, device="cuda", dtype=[F32, BF16, F16][i % 3]) for i, t in enumerate(ts)]
        check(gradients.clip_gradients(ts, bound, out=outs), ts)
        for t, o in zip(ts, outs):
            check_scaled(o, t, norm, bound)
        own = [t.clone() for t in ts]
        check(gradients.clip_gradients(own, bound), ts)
        for t, o in zip(ts, own):
            check_scaled(o, t, norm, bound)
            assert bound < norm or torch.equal(t, o)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("start", [1, 2, 3, 5, 7])
@pytest.mark.parametrize("n", [1, 6, 17, 20000])
def test_tensors_that_start_anywhere(start, n, dtype):
    """What lies in front of and behind a tensor is neither counted nor touched."""
    from haste_b200 import gradients
    g = torch.Generator(device="cuda").manual_seed(n)
    whole = torch.randn(start + n + 9, generator=g, device="cuda").to(dtype)
    whole[:start] = float("nan")
    whole[start + n:] = float("inf")
    t = whole[start:start + n]
    check(gradients.grad_norm(t), [t])
    for other in (F32, dtype):
        for shift in (0, 1, start):
            into = torch.full((n + 20,), 3.0, device="cuda", dtype=other)
            gradients.clip_gradients(t, 0.5, out=into[shift:shift + n])
            check_scaled(into[shift:shift + n], t, norm_of([t]), 0.5)
            assert (into[:shift] == 3).all() and (into[shift + n:] == 3).all()
    before = whole.clone()
    gradients.clip_gradients(t, 0.5)
    check_scaled(t, before[start:start + n], norm_of([before[start:start + n]]), 0.5)
    assert torch.equal(whole[:start].isnan(), before[:start].isnan()) and torch.equal(whole[start + n:], before[start + n:])


@pytest.mark.parametrize("scale", [1e-30, 1e-22, 1e-15, 1e15, 1e22, 1e30, 0.0])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradients_whose_squares_leave_the_range(scale, dtype):
    from haste_b200 import gradients
    g = torch.Generator(device="cuda").manual_seed(2)
    ts = make(g, [(3000,), (77, 5)], [dtype], scale) + make(g, [(50,)], [dtype], scale * 1e-3)
    check(gradients.grad_norm(ts), ts)
    own = [t.clone() for t in ts]
    gradients.clip_gradients(own, 1.0)
    for t, o in zip(ts, own):
        check_scaled(o, t, norm_of(ts), 1.0)


def test_norms_that_are_not_finite():
    from haste_b200 import clip_grad_norm_, gradients
    for bad, after in ((float("inf"), 0.0), (float("nan"), float("nan"))):
        ts = [torch.ones(10, device="cuda"), torch.ones(5000, device="cuda", dtype=BF16)]
        ts[1][4321] = bad
        p = [torch.nn.Parameter(torch.zeros_like(t)) for t in ts]
        for q, t in zip(p, ts):
            q.grad = t.clone()
        with pytest.raises(RuntimeError, match="norm of the gradients"):
            clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
        assert all(torch.equal(q.grad, t) or bad != bad for q, t in zip(p, ts))
        norm = clip_grad_norm_(p, 1.0)
        assert norm.isinf() if bad == bad else norm.isnan()
        want = torch.full((10,), after, device="cuda")
        assert torch.equal(p[0].grad, want) or (after != after and p[0].grad.isnan().all())
        assert p[1].grad[4321].isnan()
    t = torch.full((10,), 3.0, device="cuda")
    assert torch.isfinite(gradients.clip_gradients(t, float("inf"))) and (t == 3).all()
    assert gradients.clip_gradients(t, 0.0) > 0 and not t.any()


def test_axes_in_any_order_and_refusals():
    from haste_b200 import clip_grad_norm_, gradients
    base = torch.randn(6, 5, 4, device="cuda")
    t = base.permute(2, 0, 1)
    check(gradients.grad_norm([t]), [t])
    out = torch.empty_like(t)  # keeps the strides
    gradients.clip_gradients([t], 1.0, out=[out])
    check_scaled(out, t, norm_of([t]), 1.0)
    for args, error, says in (
            (([base[:, ::2]], 1.0), ValueError, "one range of memory"),
            (([base.new_zeros(1).expand(4)], 1.0), ValueError, "one range of memory"),
            (([base.double()], 1.0), TypeError, "float32, bfloat16 and float16"),
            (([base], -1.0), ValueError, "max_norm"),
            (([base], float("nan")), ValueError, "max_norm"),
            (([base, base.view(-1)], 1.0), ValueError, "overlap"),
            (([base, base[1:]], 1.0), ValueError, "overlap"),
            (([base], 1.0, [base[0]]), ValueError, "shapes"),
            (([t], 1.0, [torch.empty(t.shape, device="cuda")]), ValueError, "lie in memory"),
            (([base], 1.0, [out, out]), ValueError, "as many"),
            (([base, out], 1.0, [out.permute(1, 2, 0), base.permute(2, 0, 1)]), ValueError, "overlap"),
            (([base, base + 1], 1.0, [base.new_empty(base.shape)] * 2), ValueError, "overlap"),
            (([base, base.cpu()], 1.0), RuntimeError, "CUDA")):
        with pytest.raises(error, match=says):
            gradients.clip_gradients(*args)
    twice = base.clone()
    check(gradients.grad_norm([base, base]), [base, base])
    both = [base, out.clone()]
    check(gradients.clip_gradients([twice, out, twice], 1.0), both)  # the same tensor, in place: once
    check_scaled(twice, base, norm_of(both), 1.0)
    shared = torch.nn.Parameter(torch.zeros(6, 5, 4, device="cuda"))
    shared.grad = base.clone()
    check(clip_grad_norm_([shared, shared, torch.nn.Parameter(torch.zeros(3, device="cuda"))], 1.0), [base])
    check_scaled(shared.grad, base, norm_of([base]), 1.0)
    assert gradients.grad_norm([]).item() == 0 and clip_grad_norm_([], 1.0).item() == 0


def test_written_gradients_are_counted_as_changed():
    from haste_b200 import gradients
    t = torch.randn(10, device="cuda")
    before = t._version
    gradients.grad_norm(t)
    assert t._version == before
    gradients.clip_gradients(t, 1.0)
    assert t._version > before


def test_in_a_graph_and_on_another_stream():
    from haste_b200 import gradients
    g = torch.Generator(device="cuda").manual_seed(3)
    ts = make(g, [(1000, 300), (7,), (513,)] * 30, [F32, BF16])
    static, outs = [torch.zeros_like(t) for t in ts], [torch.zeros_like(t, dtype=F32) for t in ts]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = gradients.clip_gradients(static, 1.0, out=outs)
    for _ in range(2):
        for s, t in zip(static, ts):
            s.copy_(t)
        graph.replay()
        check(norm, ts)
        for t, o in zip(ts, outs):
            check_scaled(o, t, norm_of(ts), 1.0)
        ts = [t * 2 for t in ts]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, b = gradients.grad_norm(ts), gradients.grad_norm(ts)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b)
    check(a, ts)


def test_more_elements_than_32_bits_count():
    from haste_b200 import gradients
    t = torch.ones((1 << 31) + 4099, device="cuda", dtype=BF16)
    t[-1] = 3.0e4
    # a thread's ones add up exactly, all else is 64 bits; 3.0e4 in bfloat16 is 29952
    want = math.sqrt(t.numel() - 1 + 29952.0 ** 2)
    assert abs(gradients.clip_gradients(t, 1.0).item() - want) <= 2 * 2.0 ** -24 * want
    assert abs(t[-1].item() - 29952 / want) <= 2.0 ** -8 and abs(t[0].item() * want - 1) <= 2.0 ** -8


def test_data_parallel_clips_what_it_has_summed():
    import haste_b200
    net = haste_b200.Stack(haste_b200.LSTM, 16, 32, num_layers=2).cuda()
    dp = haste_b200.data_parallel.attach(net)
    dp.zero_grad()
    y = net(torch.randn(5, 3, 16, device="cuda"))
    (y * 100).sum().backward()
    dp.finish()
    grads = [p.grad.clone() for p in net.parameters()]
    check(dp.clip_grad_norm_(0.5), grads)
    for p, t in zip(net.parameters(), grads):
        check_scaled(p.grad, t, norm_of(grads), 0.5)
    dp.detach()
