"""The product with bias, activation and residual (csrc/linear.cu) and its gradients, against 64 bits."""
import pytest
import torch

import comprex_b200 as cx
from comprex_b200 import ComprexError

TYPES = [torch.float32, torch.bfloat16, torch.float16]
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # unit roundoff: 24, 8 and 11 bits
SMALL = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}                 # half a subnormal step
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]
# rows, inner, outer: one token, one of everything, tile borders, odd sizes, a long sum
SIZES = [(1, 64, 128), (1, 1, 1), (2, 1024, 40), (5, 7, 3), (16, 256, 512), (17, 96, 264), (128, 64, 128), (129, 72, 136), (257, 520, 255), (100, 1001, 33), (700, 8, 16)]


def _act(u, act):
    f = torch.nn.functional
    return {None: lambda v: v * 1.0, "relu": torch.relu, "gelu": f.gelu, "gelu_tanh": lambda v: f.gelu(v, approximate="tanh"), "silu": f.silu}[act](u)


def _inputs(rows, inner, outer, dtype, device, bias=True, residual=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=gen).to(dtype).to(device)  # noqa: E731
    w = (torch.randn(outer, inner, generator=gen) / inner ** 0.5).to(dtype).to(device)
    return make(rows, inner), w, make(outer) if bias else None, make(rows, outer) if residual else None, make(rows, outer)


def _check(x, w, b, r, g, act, got, grads):
    """Elementwise bounds: sums of n products in 32 bits are off by at most n 2^-23 times the sum of magnitudes (the
    order is free), every rounding to the type by UNIT, exponentials by 2^-20; the slopes change by at most 1.2 per unit."""
    dtype = x.dtype
    unit, small = UNIT[dtype], SMALL[dtype]
    X, W, G = x.double().cpu(), w.double().cpu(), g.double().cpu()
    B = torch.zeros(w.size(0), dtype=torch.float64) if b is None else b.double().cpu()
    R = 0.0 if r is None else r.double().cpu()
    n, k, m = w.size(0), w.size(1), x.size(0)
    u = (X @ W.T + B).requires_grad_()
    a = _act(u, act)
    du, = torch.autograd.grad(a, u, G)
    u, a = u.detach(), a.detach()
    e_u = (k + 4) * 2.0 ** -23 * (X.abs() @ W.abs().T + B.abs())
    y = a + R
    bound = unit * y.abs() + small + 1.2 * e_u + 2.0 ** -20 * (u.abs() + a.abs()) + 2.0 ** -23 * y.abs()
    assert ((got.detach().double().cpu() - y).abs() <= bound).all()
    if grads is None:
        return
    dx, dw, db = (None if t is None else t.double().cpu() for t in grads)
    # du before its rounding: from u in the operands' type
    e_du = G.abs() * (1.2 * (unit * u.abs() + small + e_u) + 2.0 ** -20 * (1 + u.abs())) * (act is not None)
    if act == "relu":                   # a jump where u is within its own error of zero
        e_du = torch.where(u.abs() <= e_u, G.abs(), e_du)
    e_all = e_du + (unit * (du.abs() + e_du) + small) * (act is not None)
    if dx is not None:
        bound = e_all @ W.abs() + (n + 4) * 2.0 ** -23 * (du.abs() @ W.abs()) + unit * (du @ W).abs() + small
        assert ((dx - du @ W).abs() <= 1.01 * bound).all()
    if dw is not None:
        bound = e_all.T @ X.abs() + (m + 4) * 2.0 ** -23 * (du.abs().T @ X.abs()) + unit * (du.T @ X).abs() + small
        assert ((dw - du.T @ X).abs() <= 1.01 * bound).all()
    if db is not None:
        bound = e_du.sum(0) + (m + 4) * 2.0 ** -23 * du.abs().sum(0) + unit * du.sum(0).abs() + small
        assert ((db - du.sum(0)).abs() <= 1.01 * bound).all()


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
def test_against_64_bits(device, dtype, act, size):
    x, w, b, r, g = _inputs(*size, dtype, device)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    y = cx.linear(x, w, b, activation=act, residual=r)
    dx, dw, db, dr = torch.autograd.grad(y, leaves, g)
    assert torch.equal(dr, g)
    _check(*(t.detach() for t in leaves), g, act, y, (dx, dw, db))
    with torch.no_grad():
        assert torch.equal(cx.linear(x, w, b, activation=act, residual=r), y)


@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
def test_without_bias_or_residual(device, bias, residual):
    for act in (None, "gelu_tanh"):
        x, w, b, r, g = _inputs(33, 48, 56, torch.bfloat16, device, bias, residual)
        leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
        y = cx.linear(x, w, b, activation=act, residual=r)
        got = iter(torch.autograd.grad(y, leaves, g))
        grads = [next(got) if t is not None else None for t in (x, w, b)]
        _check(x.detach(), w.detach(), None if b is None else b.detach(), r, g, act, y, grads)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(8192, 64, 64), (64, 4096, 64), (40, 64, 5000), (2049, 1024, 1032), (1, 4096, 1024), (8, 1000, 4096), (3, 4096, 4096),
                                  (513, 4095, 130), (256, 256, 512), (300, 2048, 256)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_larger_sizes(size, dtype):
    for act in (None, "silu"):
        x, w, b, r, g = _inputs(*size, dtype, "cuda")
        leaves = [t.requires_grad_() for t in (x, w, b)]
        y = cx.linear(x, w, b, activation=act, residual=r)
        grads = torch.autograd.grad(y, leaves, g)
        _check(*(t.detach() for t in leaves), r, g, act, y, grads)
        again = cx.linear(x, w, b, activation=act, residual=r)
        assert torch.equal(again, y) and all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(again, leaves, g), grads))


def test_memory_orders(device):
    """Rows that lie apart, transposed and expanded operands, a gradient of zero stride, more dimensions."""
    gen = torch.Generator().manual_seed(1)
    make = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16).to(device)  # noqa: E731
    wide_x, wide_w, wide_r = make(20, 3, 100), make(50, 90), make(60, 77)
    x, w, r, b = wide_x[:, :, 8:72], wide_w[::2, 16:80], wide_r[:, 3:28], make(50)[::2]
    y = cx.linear(x, w, b, residual=r.view(20, 3, 25))
    assert y.shape == (20, 3, 25)
    assert torch.equal(y.view(60, 25), cx.linear(x.reshape(60, 64).contiguous(), w.contiguous(), b.contiguous(), residual=r.contiguous()))
    assert torch.equal(cx.linear(x.reshape(60, 64), w.T.contiguous().T, b), cx.linear(x.reshape(60, 64), w, b))
    one = make(1, 64).expand(60, 64)
    assert torch.equal(cx.linear(one, w), cx.linear(one.contiguous(), w))
    # off a 16-byte boundary
    odd = make(60 * 64 + 1)[1:].view(60, 64)
    assert torch.equal(cx.linear(odd, w), cx.linear(odd.clone(), w))
    xr, wr = x.detach().requires_grad_(), w.detach().requires_grad_()
    ones = torch.autograd.grad(cx.linear(xr, wr, activation="silu").sum(), (xr, wr))
    full = torch.autograd.grad(cx.linear(xr, wr, activation="silu"), (xr, wr), torch.ones(20, 3, 25, dtype=x.dtype, device=device))
    assert all(torch.equal(a, c) for a, c in zip(ones, full))


def test_gradient_against_differences(device):
    """Central differences in 32 bits; the step's error is h^2 times a third derivative below 3, the sums' 2^-20 / h."""
    x, w, b, r, g = _inputs(6, 10, 8, torch.float32, device)
    for act in ("gelu", "gelu_tanh", "silu"):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        grads = torch.autograd.grad(cx.linear(*leaves, activation=act, residual=r), leaves, g)
        for leaf, grad in zip(leaves, grads):
            way = torch.randn_like(leaf)
            h = 1e-2
            with torch.no_grad():
                high, low = ((cx.linear(*(t + s * h * way if t is leaf else t for t in leaves), activation=act, residual=r).double() * g.double()).sum() for s in (1, -1))
            want = ((high - low) / (2 * h)).item()
            size = g.abs().sum().item()
            assert abs((grad.double() * way.double()).sum().item() - want) <= size * (3 * h * h * way.abs().max().item() ** 3 * 10 + 2.0 ** -20 / h * 4)


def test_empty_and_special_values(device):
    x, w, b, _, _ = _inputs(4, 16, 24, torch.float16, device)
    assert cx.linear(x[:0], w, b).shape == (0, 24)
    leaves = [t.requires_grad_() for t in (x[:0].clone(), w, b)]
    dx, dw, db = torch.autograd.grad(cx.linear(*leaves, activation="relu").sum(), leaves)
    assert dx.shape == (0, 16) and not dw.any() and not db.any()
    bad = x.detach().clone()
    bad[2, 5] = float("nan")
    for act in ACTS:
        y = cx.linear(bad, w.detach(), activation=act)
        assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3]]).all()


@pytest.mark.gpu
def test_on_another_stream_and_without_a_gradient_for_all():
    x, w, b, r, g = _inputs(300, 256, 128, torch.bfloat16, "cuda")
    want = cx.linear(x, w, b, activation="gelu_tanh", residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cx.linear(x, w, b, activation="gelu_tanh", residual=r)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    for only in range(3):
        leaves = [t.clone().requires_grad_(i == only) for i, t in enumerate((x, w, b))]
        part, = torch.autograd.grad(cx.linear(*leaves, activation="silu"), [leaves[only]], g)
        every = [t.clone().requires_grad_() for t in (x, w, b)]
        assert torch.equal(part, torch.autograd.grad(cx.linear(*every, activation="silu"), every, g)[only])


def test_refusals(device):
    x, w, b, r, _ = _inputs(4, 16, 24, torch.bfloat16, device)
    with pytest.raises(ValueError):
        cx.linear(x, w, activation="tanh")
    for bad in (dict(x=x.float()), dict(x=x[:, :8]), dict(weight=w[0]), dict(bias=b[:3]), dict(residual=r[:2]), dict(bias=b.float()), dict(residual=r.half())):
        with pytest.raises(ComprexError):
            cx.linear(**(dict(x=x, weight=w, bias=b, residual=r) | bad))
    with pytest.raises(ComprexError):
        cx.linear(x.double(), w.double())
    with pytest.raises(ComprexError):
        cx.linear(x, w[:, :0].expand(24, 0))


@pytest.mark.parametrize("dtype", TYPES)
def test_the_negative_bit(device, dtype):
    """A tensor whose sign is only noted (an imaginary part of a conjugate, say) counts with its sign."""
    x, w, b, r, g = _inputs(9, 24, 16, dtype, device)
    y = cx.linear(-x, -w, -b, activation="silu", residual=-r)
    noted = [torch._neg_view(t) for t in (x, w, b, r)]
    assert torch.equal(cx.linear(noted[0], noted[1], noted[2], activation="silu", residual=noted[3]), y)
    grads = []
    for s, up in ((lambda t: -t, -g), (torch._neg_view, torch._neg_view(g))):
        leaves = [s(t.clone()).detach().requires_grad_() for t in (x, w, b, r)]
        grads.append(torch.autograd.grad(cx.linear(*leaves[:3], activation="silu", residual=leaves[3]), leaves, up))
    assert all(torch.equal(p.resolve_neg(), q.resolve_neg()) for p, q in zip(*grads))


def test_forward_mode_is_refused(device):
    """A tangent is not dropped in silence: there is no forward-mode derivative."""
    x, w, b, r, g = _inputs(4, 16, 24, torch.float32, device)
    with torch.autograd.forward_ad.dual_level():
        for i in range(4):
            args = [torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate((x, w, b, r))]
            with pytest.raises(ComprexError, match="forward-mode"):
                cx.linear(*args[:3], residual=args[3])
        leaf = x.clone().requires_grad_()
        up = torch.autograd.forward_ad.make_dual(g, torch.ones_like(g))
        with pytest.raises(ComprexError, match="forward-mode"):
            torch.autograd.grad(cx.linear(leaf, w, b), leaf, up)


def test_tracing_is_refused(device):
    """A trace sees outputs being allocated, and no kernel: what it plays back would be memory that nobody wrote."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w, _, _, _ = _inputs(4, 16, 24, torch.float32, device)
    h, t = x[:, :16], torch.zeros(4, dtype=torch.int64, device=device)
    for f in (lambda a: cx.linear(a, w), lambda a: cx.linear_cross_entropy(a, w, t)):
        with pytest.raises(ComprexError, match="trace"):
            torch.jit.trace(f, (h,), check_trace=False)
        with pytest.raises(ComprexError, match="trace"):
            make_fx(f)(h)
    assert torch.isfinite(cx.linear(x, w)).all()

    def back(a):
        return torch.autograd.grad(y, leaf, a)[0]
    leaf = x.clone().requires_grad_()
    y = cx.linear(leaf, w)
    with pytest.raises(ComprexError, match="trace"):
        make_fx(back)(torch.ones_like(y))


def _without_memory(device):
    """Tensors that have no memory of their own to read, and how a call meets them."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    x, w, b, r, g = _inputs(4, 16, 16, torch.float32, device)
    t = torch.zeros(4, dtype=torch.int64, device=device)
    mode = FakeTensorMode()

    def faked(call):
        def f():
            with mode:
                call(*(mode.from_tensor(v) for v in (x, w, t)))
        return f

    def in_the_mode(call):
        def f():
            with mode:
                call(x, w, t)
        return f

    def zero(call):
        return lambda: call(torch._efficientzerotensor((4, 16), device=device), w, t)

    def mapped(call):
        return lambda: torch.vmap(lambda a: call(a[None], w, t[:1]))(x)

    def differentiated(call):
        return lambda: torch.func.grad(lambda a: call(a, w, t).sum())(x)
    return [k(call) for k in (faked, in_the_mode, zero, mapped, differentiated)
            for call in (lambda a, c, i: cx.linear(a, c), lambda a, c, i: cx.linear(x, c, residual=a),
                         lambda a, c, i: cx.linear_cross_entropy(a, c, i))]


@pytest.mark.parametrize("which", range(15))
def test_tensors_without_memory_are_refused(device, which):
    with pytest.raises(ComprexError):
        _without_memory(device)[which]()


def test_backward_without_memory_is_refused(device):
    from torch._subclasses.fake_tensor import FakeTensorMode
    x, w, _, _, _ = _inputs(4, 16, 16, torch.float32, device)
    leaf = x.clone().requires_grad_()
    t = torch.zeros(4, dtype=torch.int64, device=device)
    for y in (cx.linear(leaf, w), cx.linear_cross_entropy(leaf, w, t, reduction="none")):
        with pytest.raises(ComprexError), FakeTensorMode(allow_non_fake_inputs=True):
            torch.autograd.grad(y, leaf, torch.ones(y.shape, device=device), retain_graph=True)
        # no gradient at all, without memory for it
        got, = torch.autograd.grad(y, leaf, torch._efficientzerotensor(tuple(y.shape), device=device))
        assert not got.any()


@pytest.mark.parametrize("rows", [1, 300])
def test_activations_in_32_bits_to_their_ends(device, rows):
    """float32 values and slopes relative to themselves, down to where they leave the normal numbers: an exponential of an exact
    argument is good to a few units of 2^-24, one of a rounded argument y to |y| more of them."""
    f = torch.nn.functional
    u = torch.cat((torch.linspace(-100, 100, 4001), torch.linspace(-6, 6, 999), torch.tensor([-1e-30, 0.0, 1e-30, -1e30, 1e30])))
    u = u.double().float()
    u64 = u.double().requires_grad_()
    x = torch.ones(rows, 1, device=device).requires_grad_()
    w = u[:, None].to(device)
    z2 = 2 * 0.7978845608028654 * (u64.detach() + 0.044715 * u64.detach() ** 3)
    for act, value, off in (("silu", u64 * torch.sigmoid(u64), 8.0),
                            # u (1 + tanh z) / 2 = u sigmoid(2 z), without the sum's cancellation; the argument has six roundings
                            ("gelu_tanh", u64 * torch.sigmoid(2 * 0.7978845608028654 * (u64 + 0.044715 * u64 ** 3)), 8.0 + 6 * z2.abs())):
        slope, = torch.autograd.grad(value.sum(), u64, retain_graph=True)
        y = cx.linear(x, w, activation=act)
        # one output of one row at a time: dx is its slope times u, so take the bias's gradient
        b = torch.zeros(u.numel(), device=device).requires_grad_()
        db, = torch.autograd.grad(cx.linear(x[:1].detach(), w, b, activation=act), b, torch.ones(1, u.numel(), device=device))
        value = value.detach()
        off = torch.as_tensor(off) * 2.0 ** -24
        assert ((y.detach().double().cpu() - value).abs() <= off * value.abs() + 1e-36).all(), act
        # the slope is a sum of two terms that cancel: relative to both
        gate = torch.sigmoid(u64.detach() if act == "silu" else z2)
        inner = u64.detach() if act == "silu" else z2 + 2 * 2 * 0.7978845608028654 * 0.044715 * u64.detach() ** 3
        terms = gate + (inner * gate * (1 - gate)).abs()
        finite = u64.detach().abs() < 1e18            # (beyond, the cube leaves 32 bits, here as anywhere)
        assert ((db.double().cpu() - slope).abs() <= 3 * off * terms + 1e-36)[finite].all(), act


@pytest.mark.parametrize("low", [torch.bfloat16, torch.float16])
def test_autocast(device, low):
    """Products are in autocast's type, as torch's; what is added to them keeps its own."""
    x, w, b, r, _ = _inputs(20, 32, 24, torch.float32, device)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
    cast = [t.clone().to(low).requires_grad_() for t in (x, w, b)]
    with torch.autocast(device, dtype=low):
        y = cx.linear(*leaves[:3], activation="silu", residual=leaves[3])
        z = cx.linear(*leaves[:3], activation="silu", residual=leaves[3].to(low))
        assert cx.linear(x, w).dtype == torch.nn.functional.linear(x, w).dtype == low
    assert y.dtype == torch.float32 and z.dtype == low
    inner = cx.linear(*cast, activation="silu")
    assert torch.equal(y, inner + r) and torch.equal(z, cx.linear(*cast, activation="silu", residual=r.to(low)))
    g = torch.randn(20, 24, generator=torch.Generator().manual_seed(2)).to(device)
    got, want = torch.autograd.grad(y, leaves, g), torch.autograd.grad(inner, cast, g.to(low))
    assert all(p.dtype == torch.float32 and torch.equal(p, q.float()) for p, q in zip(got, want)) and torch.equal(got[3], g)
    with torch.autocast(device, enabled=False):
        assert cx.linear(x, w).dtype == torch.float32
    with torch.autocast(device, dtype=low), pytest.raises(ComprexError):
        cx.linear(x.double(), w.double())


def _with_failing_calls(names, f):
    """``f()`` while these native calls return an error."""
    import ctypes as C
    from comprex_b200 import _lib
    lib, host = _lib.load(), _lib.host()
    every = ("cx_linear_workspace_bytes", "cx_linear_forward", "cx_linear_backward", "cx_vocab_loss_workspace_bytes", "cx_vocab_loss_forward",
             "cx_vocab_loss_backward", "cx_last_error")
    fails = C.CFUNCTYPE(C.c_int, C.c_int, C.c_void_p, C.c_void_p)(lambda *a: -7)
    address = [C.cast(fails if n in names else getattr(lib, n), C.c_void_p).value for n in every]
    try:
        host.bind_operators(ComprexError, *address)
        f()
    finally:
        host.bind_operators(ComprexError, *(C.cast(getattr(lib, n), C.c_void_p).value for n in every))


def test_errors_of_native_calls(device):
    """A call that fails below is the package's error, forward, in a training step and in its backward pass."""
    x, w, _, _, g = _inputs(4, 16, 24, torch.float32, device)
    t = torch.zeros(4, dtype=torch.int64, device=device)
    leaf = x.clone().requires_grad_()
    calls = [lambda a: cx.linear(a, w, activation="silu"), lambda a: cx.linear_cross_entropy(a, w, t, reduction="none")]

    def forward():
        for f in calls:
            for a in (x, leaf):
                with pytest.raises(ComprexError, match=r"forward failed: .*\(rc=-7\)"):
                    f(a)
    _with_failing_calls(("cx_linear_forward", "cx_vocab_loss_forward"), forward)

    def backward():
        for f in calls:
            y = f(leaf)
            with pytest.raises(ComprexError, match=r"backward failed: .*\(rc=-7\)"):
                torch.autograd.grad(y.sum(), leaf)
    _with_failing_calls(("cx_linear_backward", "cx_vocab_loss_backward"), backward)
    assert torch.isfinite(torch.autograd.grad(calls[0](leaf).sum(), leaf)[0]).all()


def test_many_outputs_in_32_bits(device):
    """More tiles of columns than a grid's second dimension has."""
    n = 64 * 65535 + 70
    x = torch.tensor([[0.5], [-2.0], [3.0], [1.0], [0.25]], device=device)
    w = torch.arange(n, dtype=torch.float32, device=device)[:, None]
    assert torch.equal(cx.linear(x, w), x * w.T)


@pytest.mark.parametrize("dtype", TYPES)
def test_zeros_times_what_is_no_number(device, dtype):
    """Gradients are sums of products: zero times infinity is no number on either back end, as in torch."""
    x, w, _, _, g = _inputs(6, 16, 24, dtype, device)
    g[2], g[:, 5] = 0.0, 0.0
    x[2, 3], x[4, 1], w[5, 2], w[7, 9] = float("inf"), float("nan"), float("inf"), float("nan")
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    got = torch.autograd.grad(cx.linear(*leaves), leaves, g)
    want = g.float() @ w.float(), g.float().T @ x.float()
    assert all(torch.equal(torch.isnan(a), torch.isnan(b)) for a, b in zip(got, want))


def test_saved_tensors_that_come_back_changed(device):
    """Hooks may keep what is saved in another order; what comes back as something else is refused, not read as if it were the same."""
    from torch.autograd.graph import saved_tensors_hooks
    x, w, b, _, g = _inputs(6, 32, 24, torch.bfloat16, device)
    t = torch.arange(6, device=device)
    leaves = [v.requires_grad_() for v in (x, w, b)]
    calls = [lambda: cx.linear(*leaves, activation="gelu"), lambda: cx.linear(*leaves),
             lambda: cx.linear_cross_entropy(x, w, t, reduction="none")]
    for f in calls:
        y = f()
        up = torch.ones_like(y)
        want = torch.autograd.grad(y, leaves, up, allow_unused=True)

        def spread(v):                         # the same numbers, further apart
            return torch.stack((v, v), -1)[..., 0]
        with saved_tensors_hooks(lambda v: v, spread):
            y = f()
        got = torch.autograd.grad(y, leaves, up, allow_unused=True)
        assert all(p is None or torch.equal(p, q) for p, q in zip(got, want))
        for other in (lambda v: v[:2], lambda v: v.double(), lambda v: v[None], lambda v: v.float() + 0, lambda v: v.to("cpu") if v.is_cuda else v[..., :1]):
            n = 0

            def one(v, which):
                nonlocal n
                n += 1
                return other(v) if n - 1 == which else v
            for which in range(5):
                n = 0
                with saved_tensors_hooks(lambda v: v, lambda v: one(v, which)):
                    y = f()
                changed = False
                try:
                    got = torch.autograd.grad(y, leaves, up, allow_unused=True)
                except (ComprexError, RuntimeError):
                    changed = True
                # either refused, or what came back was the same after all (nothing left to change, a number in float32 already)
                assert changed or all(p is None or torch.equal(p, q) for p, q in zip(got, want)), which


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(300, 700, 1000), (1030, 67, 515), (4, 4096, 4096), (5, 3000, 130)])
def test_larger_sizes_in_32_bits(size):
    """Many tiles of the CUDA cores' product in all three layouts, and few rows of large weights."""
    for act in (None, "gelu"):
        x, w, b, r, g = _inputs(*size, torch.float32, "cuda")
        leaves = [t.requires_grad_() for t in (x, w, b)]
        y = cx.linear(x, w, b, activation=act, residual=r)
        grads = torch.autograd.grad(y, leaves, g)
        _check(*(t.detach() for t in leaves), r, g, act, y, grads)
        again = cx.linear(x, w, b, activation=act, residual=r)
        assert torch.equal(again, y) and all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(again, leaves, g), grads))
