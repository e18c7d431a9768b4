"""MXFP4 entry points on operands whose rows the kernels cannot read as they lie: the calls copy them, and give what the copy gives."""
import pytest
import torch

from sglang_amd import mxfp4

pytestmark = pytest.mark.gpu


def _random(shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def test_expanded_operands(dev):
    """One row of codes for all rows: a row stride of zero."""
    q, s = mxfp4.per_token_group_quant_mxfp4(_random((1, 288)))
    w, ws = mxfp4.quant_weight_mxfp4(_random((72, 288), seed=1))
    one = mxfp4.w4a4_mxfp4_matmul(q, w, s, ws)
    for m in (2, 8, 70):
        got = mxfp4.w4a4_mxfp4_matmul(q.expand(m, -1), w, s.expand(m, -1), ws)
        assert torch.equal(got, mxfp4.w4a4_mxfp4_matmul(q.repeat(m, 1), w, s.repeat(m, 1), ws))
        assert torch.equal(got, got[:1].expand(m, -1)) and (m > 16 or torch.equal(got[:1], one))
    x = _random((5, 288), seed=2)
    for rows in (x, x[:1], x.expand(3, 5, 288), x[:1].expand(4, 288)):
        got = mxfp4.w4a4_mxfp4_linear(rows, w[:1].expand(16, -1), ws[:1].expand(16, -1))
        assert torch.equal(got, mxfp4.w4a4_mxfp4_linear(rows.contiguous(), w[:1].repeat(16, 1), ws[:1].repeat(16, 1)))


def _shifted(t, elements):
    """t's values in rows that start `elements` elements behind a multiple of 16 bytes, a multiple of 16 bytes apart."""
    wide = torch.zeros((t.shape[0], t.shape[1] + 64), dtype=t.dtype, device=t.device)
    wide[:, elements:elements + t.shape[1]] = t
    view = wide[:, elements:elements + t.shape[1]]
    assert view.data_ptr() % 16 != 0 and view.stride(0) * view.element_size() % 16 == 0
    return view


def _experts(e, h, i):
    (w1, s1), (w2, s2) = mxfp4.quant_weight_mxfp4(_random((e, 2 * i, h), seed=3) * 0.1), mxfp4.quant_weight_mxfp4(_random((e, h, i), seed=4) * 0.1)
    return w1, w2, s1, s2


# 20 rows: both ways of a linear are a quantisation and a product then
X, W, E = (20, 288), (72, 288), (5, 288, 96)


def _calls(place):
    """Every entry point, its operand laid out by `place`."""
    w, ws = mxfp4.quant_weight_mxfp4(_random(W, seed=1))
    q, s = mxfp4.per_token_group_quant_mxfp4(_random(X))
    w1, w2, s1, s2 = _experts(*E)
    weights, ids = torch.rand((X[0], 2), generator=torch.Generator().manual_seed(5)).cuda(), (torch.arange(2 * X[0], device="cuda") % E[0]).view(X[0], 2)
    x, gate_up = _random(X), _random((X[0], 2 * X[1]), torch.float16, seed=6)
    return [("quant", lambda t: mxfp4.per_token_group_quant_mxfp4(t), place(x)), ("quant32", lambda t: mxfp4.per_token_group_quant_mxfp4(t), place(x.float())),
            ("silu", lambda t: mxfp4.per_token_group_quant_mxfp4(t, True), place(gate_up)),
            ("dequant", lambda t: mxfp4.mxfp4_dequant(t, s, torch.float16), place(q)),
            ("matmul", lambda t: mxfp4.w4a4_mxfp4_matmul(t, w, s, ws), place(q)), ("weight", lambda t: mxfp4.w4a4_mxfp4_matmul(q, t, s, ws), place(w)),
            ("linear", lambda t: mxfp4.w4a4_mxfp4_linear(t, w, ws), place(x)),
            ("experts", lambda t: mxfp4.fused_experts_mxfp4(t, w1, w2, weights, ids, s1, s2), place(x))]


def _equal(a, b):
    a, b = (t if isinstance(t, tuple) else (t,) for t in (a, b))
    return len(a) == len(b) and all(torch.equal(t, u) for t, u in zip(a, b))


@pytest.mark.parametrize("name", ["quant", "quant32", "silu", "dequant", "matmul", "weight", "linear", "experts"])
def test_rows_that_start_anywhere(dev, name):
    """Operands that do not start at a multiple of 16 bytes: a view of other rows, and contiguous memory; eager and traced."""
    want, got = [], []
    for place in (lambda t: t, lambda t: _shifted(t, 3), lambda t: _shifted(t.flatten()[None], 1).view(t.shape)):
        fn, t = next((f, t) for n, f, t in _calls(place) if n == name)
        want.append(fn(t))
        torch._dynamo.reset()
        got.append(torch.compile(fn, backend="aot_eager", fullgraph=True)(t))
    assert all(_equal(w, want[0]) for w in want), "eager"
    assert all(_equal(g, want[0]) for g in got), "traced"


def test_traced_once_for_both_alignments(dev):
    """One trace serves operands of the same shape and strides at any address."""
    w, ws = mxfp4.quant_weight_mxfp4(_random(W, seed=1))
    x = _random(X)
    wide = torch.zeros((X[0], X[1] + 64), dtype=x.dtype, device=dev)
    fn = torch.compile(lambda t: mxfp4.w4a4_mxfp4_linear(t, w, ws), backend="aot_eager", fullgraph=True)
    for at in (0, 8, 5, 16, 1):
        wide[:, at:at + X[1]] = x
        assert torch.equal(fn(wide[:, at:at + X[1]]), mxfp4.w4a4_mxfp4_linear(x, w, ws)), at


def test_inplace_experts_of_a_view(dev):
    w1, w2, s1, s2 = _experts(*E)
    x = _random(X)
    weights, ids = torch.rand((X[0], 2), generator=torch.Generator().manual_seed(5)).cuda(), (torch.arange(2 * X[0], device="cuda") % E[0]).view(X[0], 2)
    want = mxfp4.fused_experts_mxfp4(x, w1, w2, weights, ids, s1, s2)
    view = _shifted(x, 3)
    got = mxfp4.fused_experts_mxfp4(view, w1, w2, weights, ids, s1, s2, inplace=True)
    assert got.data_ptr() == view.data_ptr() and torch.equal(view, want)


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.float16, torch.float8_e4m3fn, torch.float8_e5m2])
def test_weights_of_any_float_type(dev, dtype):
    """What the kernel does not read itself goes through float32, which holds every 8-bit value."""
    w = (_random((3, 40, 96), torch.float32) * 3).to(dtype)
    for t in (w, w[1]):
        got, want = mxfp4.quant_weight_mxfp4(t), mxfp4.quant_weight_mxfp4(t.float())
        assert _equal(got, want)
    with pytest.raises(RuntimeError):
        mxfp4.quant_weight_mxfp4(torch.zeros((8, 32), dtype=torch.int32, device=dev))


@pytest.mark.parametrize("m", [1, 5, 21, 70])
def test_traced_feed_forward_with_odd_rows(dev, m):
    """Scale words of a number of rows that is no multiple of four are a view of a padded buffer; tracing hands it from call to call."""
    up, ups = mxfp4.quant_weight_mxfp4(_random((2 * 96, 288), seed=1))
    down, downs = mxfp4.quant_weight_mxfp4(_random((288, 96), seed=2))

    def forward(x):
        q, s = mxfp4.per_token_group_quant_mxfp4(x)
        h = mxfp4.w4a4_mxfp4_matmul(q, up, s, ups)
        q, s = mxfp4.per_token_group_quant_mxfp4(h, fuse_silu_and_mul=True)
        return mxfp4.w4a4_mxfp4_linear(q, down, downs, input_scale=s), mxfp4.mxfp4_dequant(q, s, torch.float32)

    x = _random((m, 288), seed=m)
    torch._dynamo.reset()
    for got, want in zip(torch.compile(forward, backend="aot_eager", fullgraph=True)(x), forward(x)):
        assert torch.equal(got, want)


def test_operands_that_want_gradients(dev):
    """There are none: the results are those of detached operands and require no gradient."""
    w, ws = mxfp4.quant_weight_mxfp4(_random(W, seed=1))
    w1, w2, s1, s2 = _experts(*E)
    x = _random(X)
    weights, ids = torch.rand((X[0], 2), generator=torch.Generator().manual_seed(5)).cuda(), (torch.arange(2 * X[0], device="cuda") % E[0]).view(X[0], 2)
    wants = x.clone().requires_grad_()
    for fn in (lambda t: mxfp4.per_token_group_quant_mxfp4(t)[0], lambda t: mxfp4.w4a4_mxfp4_linear(t, w, ws),
               lambda t: mxfp4.fused_experts_mxfp4(t, w1, w2, weights, ids, s1, s2)):
        got = fn(wants)
        assert torch.equal(got, fn(x)) and not got.requires_grad


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k", [(2, 288), (4, 4096), (16, 160), (20, 288), (70, 1056)])
def test_rows_that_are_not_finite_stay_alone_in_a_linear(dev, m, k, dtype):
    """Quantised inside (up to 16 rows) or in front of the product."""
    w, ws = mxfp4.quant_weight_mxfp4(_random((72, k), seed=1))
    x = _random((m, k), dtype)
    clean = mxfp4.w4a4_mxfp4_linear(x, w, ws)
    bad = x.clone()
    bad[1, k - 1], bad[m // 2, 0] = float("nan"), float("-inf")
    got = mxfp4.w4a4_mxfp4_linear(bad, w, ws)
    rest = torch.tensor([r not in (1, m // 2) for r in range(m)], device=dev)
    assert torch.equal(got[rest], clean[rest]) and got[1].isnan().all() and got[m // 2].isnan().all()


def test_threads_and_streams_at_once(dev):
    """Four threads, each on a stream of its own, through the calls that take scratch memory."""
    import threading

    w, ws = mxfp4.quant_weight_mxfp4(_random(W, seed=1))
    w1, w2, s1, s2 = _experts(*E)
    xs = [_random((21 + 10 * j, X[1]), seed=10 + j) for j in range(4)]
    weights = [torch.rand((x.shape[0], 2), generator=torch.Generator().manual_seed(5)).cuda() for x in xs]
    ids = [(torch.arange(2 * x.shape[0], device=dev) % E[0]).view(-1, 2) for x in xs]

    def step(j):
        return mxfp4.w4a4_mxfp4_linear(xs[j], w, ws), mxfp4.fused_experts_mxfp4(xs[j], w1, w2, weights[j], ids[j], s1, s2)

    want = [step(j) for j in range(4)]
    torch.cuda.synchronize()
    wrong = []

    def work(j):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got = [step(j) for _ in range(50)]
        stream.synchronize()
        wrong.extend((j, i) for i, g in enumerate(got) if not _equal(g, want[j]))

    threads = [threading.Thread(target=work, args=(j,)) for j in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
