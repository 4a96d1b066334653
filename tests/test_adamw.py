"""AdamW over many tensors (csrc/adamw.cu): against the formula in 64 bits, its 8-bit states, its refusals."""
import math

import numpy as np
import pytest
import torch

import comprex_b200 as cx
from comprex_b200 import ComprexError

SIZES = [1, 3, 255, 256, 257, 1000, 4096, 10007]
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
EPS32 = 2.0 ** -24
ROUND = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # of the stored copy


def _params(dtype, device, sizes=SIZES, seed=0, shift=0):
    """Leaves of the given sizes; ``shift``: start them that many elements off a 16-byte boundary."""
    gen = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        store = torch.zeros(n + shift, dtype=dtype, device=device)
        store[shift:] = torch.randn(n, generator=gen).to(dtype)
        out.append(torch.nn.Parameter(store[shift:]))
    return out


def _set_grads(params, seed, scale=1e-2):
    gen = torch.Generator().manual_seed(seed)
    for p in params:
        p.grad = (torch.randn(p.numel(), generator=gen) * scale).to(p.dtype).to(p.device).view(p.size())


def _formula(p, m, v, g, t, lr, betas, eps, weight_decay):
    b1, b2 = betas
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = (1 - lr * weight_decay) * p - lr * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
    return p, m, v


def _weights(opt, params):
    flat = opt.flat_state().get("master")
    if flat is None:
        return [p.detach().double().cpu().flatten() for p in params]
    return [flat[a:a + n].double().cpu() for a, n in opt.spans()]


def _decoded(opt, name):
    flat = opt.flat_state()
    x = flat[name].cpu().float().double().view(-1, 256) * flat[name + "_scale"].cpu().double()[:, None]
    return [x.flatten()[a:a + n] for a, n in opt.spans()]


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("dtype", TYPES)
def test_32_bit_states_against_the_formula(device, dtype, shift):
    params = _params(dtype, device, shift=shift)
    opt = cx.AdamW(params, state_bits=32, **HYPER)
    want = [(p.detach().double().cpu(), 0.0, 0.0) for p in params]
    steps = 5
    for t in range(1, steps + 1):
        _set_grads(params, seed=t)
        want = [_formula(*w, p.grad.double().cpu(), t, **HYPER) for w, p in zip(want, params)]
        opt.step()
    flat = opt.flat_state()
    for got, p, (wp, wm, wv), (a, n) in zip(_weights(opt, params), params, want, opt.spans()):
        # per step: two roundings of p, and a change of at most ~10 lr (a cancelled m over a small v) with eight roundings
        assert (got - wp).abs().max() <= steps * EPS32 * (2 * wp.abs().max() + 10 * HYPER["lr"] * 8) + 1e-7
        # per step three roundings of sums of magnitudes that the largest gradient bounds
        assert (flat["exp_avg"][a:a + n].double().cpu() - wm).abs().max() <= 4 * steps * EPS32 * 0.06
        assert ((flat["exp_avg_sq"][a:a + n].double().cpu() - wv).abs() <= 6 * steps * EPS32 * wv + 1e-30).all()
        # the tensor is the rounded weight
        assert torch.equal(p.detach().cpu(), got.float().to(dtype))
    # the gaps between the tensors stay empty
    gap = torch.ones(flat["exp_avg"].numel(), dtype=torch.bool)
    for a, n in opt.spans():
        gap[a:a + n] = False
    assert not flat["exp_avg"].cpu()[gap].any() and not flat["exp_avg_sq"].cpu()[gap].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_8_bit_states_hold_the_moments(device, dtype):
    params = _params(dtype, device)
    opt = cx.AdamW(params, state_bits=8, seed=3, **HYPER)
    want = [p.detach().double().cpu() for p in params]
    held_m, held_r = ([torch.zeros_like(w) for w in want] for _ in range(2))
    for t in range(1, 6):
        _set_grads(params, seed=t)
        new = [_formula(w, m, r * r, p.grad.double().cpu(), t, **HYPER) for w, m, r, p in zip(want, held_m, held_r, params)]
        opt.step()
        want = _weights(opt, params)
        for (wp, _, _), got in zip(new, want):
            assert (got - wp).abs().max() <= EPS32 * (2 * wp.abs().max() + 10 * HYPER["lr"] * 8) + 1e-7
        held_m, held_r = _decoded(opt, "exp_avg"), _decoded(opt, "exp_avg_rms")
        flat = opt.flat_state()
        for i, (_, m, v) in enumerate(new):
            block = np.arange(m.numel()) // 256 + opt.spans()[i][0] // 256
            for got, exact, scale in ((held_m[i], m, flat["exp_avg_scale"]), (held_r[i], v.sqrt(), flat["exp_avg_rms_scale"])):
                s = scale.cpu().double()[block]
                # one step of three bits of mantissa, or in the subnormals two of theirs (cut at random, then rounded)
                assert ((got - exact).abs() <= exact.abs() * (2.0 ** -3 + 1e-6) + s * 2.0 ** -9 * 1.5).all()
                assert ((exact.abs() / s) < 256.01).all()
            assert ((held_r[i] > 0) == (v > 0)).all()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.gpu
def test_cuda_agrees_with_host(dtype, bits):
    """States bit for bit.  The kernel takes the quotient of the step from the hardware's approximate reciprocal: weights
    within a few roundings of the step, which is at most 10 lr, and their own."""
    made = {}
    for device in ("cpu", "cuda"):
        params = _params(dtype, device)
        opt = cx.AdamW(params, state_bits=bits, seed=7, **HYPER)
        for t in range(4):
            _set_grads(params, seed=t)
            opt.step()
        made[device] = {k: t.cpu() for k, t in opt.flat_state().items()}
        made[device]["weights"] = torch.cat(_weights(opt, params))
    host, cuda = made["cpu"], made["cuda"]
    for k in host:
        if k.startswith("exp_avg"):
            assert torch.equal(host[k].view(torch.uint8), cuda[k].view(torch.uint8)), k
    assert ((host["weights"] - cuda["weights"]).abs() <= 4 * (EPS32 * 2 * host["weights"].abs() + 2.0 ** -21 * 10 * HYPER["lr"])).all()


def test_rounding_is_unbiased(device):
    """The same gradient everywhere: the mean of n states rounded at random is the moment itself."""
    n, g = 1 << 16, 0.01
    p = torch.nn.Parameter(torch.zeros(n, device=device))
    opt = cx.AdamW([p], state_bits=8, lr=0.0, betas=(0.9, 0.99), weight_decay=0.0)
    grad = torch.full((n,), g, device=device)
    grad[::256] = 0.0137         # the largest of each block, so that the others lie inside a step
    p.grad = grad
    opt.step()
    keep = torch.arange(n) % 256 != 0
    for name, exact in (("exp_avg", 0.1 * g), ("exp_avg_rms", math.sqrt(0.01) * g)):
        got = _decoded(opt, name)[0][keep]
        step = (got.max() - got.min()).item()
        assert got.min() <= exact <= got.max() and got.unique().numel() == 2
        # five standard deviations of the mean of independent roundings, and the 16 bits' own resolution
        assert abs(got.mean().item() - exact) <= step * (5 * 0.5 / math.sqrt(keep.sum().item()) + 2.0 ** -16)


def test_a_second_moment_does_not_stick(device):
    """b2 near one: the states of a block follow a gradient that has become small, though one change is below a step."""
    n = 4096
    p = torch.nn.Parameter(torch.zeros(n, device=device))
    opt = cx.AdamW([p], state_bits=8, lr=0.0, betas=(0.9, 0.98), weight_decay=0.0)
    first = torch.ones(n, device=device)
    later = torch.full((n,), 0.25, device=device)
    later[::256] = 1.0
    p.grad = first
    opt.step()
    p.grad = later
    steps = 60
    for _ in range(steps):
        opt.step()
    got = (_decoded(opt, "exp_avg_rms")[0][torch.arange(n) % 256 != 0] ** 2).mean().item()
    exact = 0.02 * 0.98 ** steps + 0.0625 * (1 - 0.98 ** steps)
    # each step adds the variance of a rounded root (at most (2^-3)^2 / 4 of v) to the mean of v, which b2 forgets again
    assert exact * 0.98 <= got <= exact * (1 + steps * 2.0 ** -8 * 1.05)


def test_groups_and_missing_gradients(device):
    a, b, c = _params(torch.float32, device, [300, 5, 700])
    opt = cx.AdamW([{"params": [a, b], "lr": 0.1, "weight_decay": 0.0}, {"params": [c], "betas": (0.5, 0.9)}], lr=0.01, weight_decay=0.5)
    hyper = [dict(lr=0.1, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)] * 2 + [dict(lr=0.01, betas=(0.5, 0.9), eps=1e-8, weight_decay=0.5)]
    want = [(p.detach().double().cpu(), torch.zeros(p.numel(), dtype=torch.float64), torch.zeros(p.numel(), dtype=torch.float64), 0) for p in (a, b, c)]
    for turn, missing in enumerate([(), (1,), (0, 2), (), (1,), ()]):
        _set_grads([a, b, c], seed=turn)
        for i, p in enumerate((a, b, c)):
            if i in missing:
                p.grad = None
                continue
            w, m, v, t = want[i]
            want[i] = (*_formula(w, m, v, p.grad.double().cpu(), t + 1, **hyper[i]), t + 1)
        opt.step()
    for p, (w, _, _, _) in zip((a, b, c), want):
        assert (p.detach().double().cpu() - w).abs().max() <= 6 * EPS32 * (2 * w.abs().max() + 10 * 0.1 * 8) + 1e-7
    opt.param_groups[0]["lr"] = 0.0
    before = a.detach().clone()
    opt.step()
    assert torch.equal(a.detach(), before)


@pytest.mark.parametrize("bits", [8, 32])
def test_checkpoint_goes_on_where_it_was(device, bits):
    def run(opt, params, steps):
        for t in steps:
            _set_grads(params, seed=t)
            opt.step()
    a = _params(torch.bfloat16, device)
    whole = cx.AdamW(a, state_bits=bits, seed=5, **HYPER)
    run(whole, a, range(4))
    b = _params(torch.bfloat16, device)
    part = cx.AdamW(b, state_bits=bits, seed=5, **HYPER)
    run(part, b, range(2))
    saved = part.state_dict()
    c = _params(torch.bfloat16, device, seed=9)
    other = cx.AdamW(c, state_bits=bits, **HYPER)
    other.load_state_dict(saved)
    run(other, c, range(2, 4))
    for x, y in zip(a, c):
        assert torch.equal(x, y)
    for k, t in whole.flat_state().items():
        assert torch.equal(t.view(torch.uint8), other.flat_state()[k].view(torch.uint8)), k


def test_memory_orders_and_other_gradients(device):
    """Channels-last weights keep their order; a gradient of another order or type is brought into the tensor's."""
    w = torch.randn(6, 4, 5, 5).to(device).to(memory_format=torch.channels_last)
    p, q = torch.nn.Parameter(w.clone(memory_format=torch.preserve_format)), torch.nn.Parameter(w.contiguous().clone())
    g = torch.randn(6, 4, 5, 5).to(device)
    p.grad, q.grad = g.contiguous(), g.contiguous()
    cx.AdamW([p], lr=0.1).step()
    cx.AdamW([q], lr=0.1).step()
    assert p.stride() != q.stride() and torch.equal(p.detach(), q.detach())


@pytest.mark.parametrize("bits", [8, 32])
def test_a_bad_gradient_spoils_its_element(device, bits):
    p = torch.nn.Parameter(torch.ones(600, device=device))
    opt = cx.AdamW([p], state_bits=bits, lr=0.1)
    g = torch.full((600,), 0.01, device=device)
    g[17], g[300] = float("nan"), float("inf")
    p.grad = g
    opt.step()
    p.grad = torch.full((600,), 0.01, device=device)
    opt.step()
    bad = ~torch.isfinite(p.detach().cpu())
    assert bad.nonzero().flatten().tolist() == [17, 300]


def test_zero_gradients_leave_zero_states(device):
    p = torch.nn.Parameter(torch.ones(300, device=device))
    opt = cx.AdamW([p], state_bits=8, lr=0.1, weight_decay=0.0)
    p.grad = torch.zeros(300, device=device)
    opt.step()
    assert torch.equal(p.detach().cpu(), torch.ones(300))
    for name in ("exp_avg", "exp_avg_rms"):
        assert not _decoded(opt, name)[0].any()


def test_refusals(device):
    p = torch.nn.Parameter(torch.zeros(4, 4, device=device))
    with pytest.raises(ValueError):
        cx.AdamW([p], state_bits=16)
    with pytest.raises(ValueError):
        cx.AdamW([p], lr=-1.0)
    with pytest.raises(ValueError):
        cx.AdamW([p], betas=(0.9, 1.0))
    with pytest.raises(ComprexError):
        cx.AdamW([p, torch.nn.Parameter(torch.zeros(4, dtype=torch.bfloat16, device=device))])
    with pytest.raises(ComprexError):
        cx.AdamW([torch.nn.Parameter(torch.zeros(4, dtype=torch.float64, device=device))])
    with pytest.raises(ComprexError):
        cx.AdamW([torch.nn.Parameter(torch.zeros(4, 8, device=device)[:, :4])])
    opt = cx.AdamW([p])
    with pytest.raises(ComprexError):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2, device=device))]})
    with pytest.raises(ComprexError):
        opt.load_state_dict(torch.optim.AdamW([p]).state_dict())
    with pytest.raises(ComprexError):
        opt.load_state_dict(cx.AdamW([p], state_bits=8).state_dict())
    opt.step()                   # no gradient anywhere: nothing moves
    assert not p.detach().any()


@pytest.mark.gpu
def test_a_step_is_not_captured():
    p = torch.nn.Parameter(torch.zeros(300, device="cuda"))
    p.grad = torch.ones(300, device="cuda")
    opt = cx.AdamW([p])
    opt.step()
    before = p.detach().clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(1, device="cuda")
        with pytest.raises(ComprexError):
            opt.step()
    opt.step()
    assert not torch.equal(p.detach(), before)


def _replaced(p, how):
    """``p.data`` as another tensor than the one that the optimizer was made for, with a gradient that fits it."""
    if how == "shorter":
        p.data = torch.zeros(4, 2, 2, 2, dtype=p.dtype, device=p.device)
    elif how == "longer":
        p.data = torch.zeros(4, 3, 2, 8, dtype=p.dtype, device=p.device)
    elif how == "shape":
        p.data = p.data.reshape(3, 4, 2, 2).clone()
    elif how == "order":
        p.data = p.data.contiguous(memory_format=torch.channels_last)
    elif how == "dimensions":
        p.data = p.data.reshape(48).clone()
    p.grad = torch.ones_like(p)


@pytest.mark.parametrize("how", ["shorter", "longer", "shape", "order", "dimensions"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_replaced_tensor_is_refused(device, dtype, how):
    """Length and order of the flat states are those of construction: a step over another tensor would leave it, or mix it up."""
    p = torch.nn.Parameter(torch.randn(4, 3, 2, 2, generator=torch.Generator().manual_seed(0)).to(device, dtype))
    opt = cx.AdamW([p], lr=0.1)
    was = p.data
    held = {k: t.clone() for k, t in opt.flat_state().items()}
    _replaced(p, how)
    before = p.detach().clone()
    for call in (opt.step, opt.refresh_master, lambda: opt.load_state_dict(cx.AdamW([torch.nn.Parameter(was.clone())]).state_dict())):
        with pytest.raises(ComprexError, match="as it was"):
            call()
    assert torch.equal(p.detach(), before)
    assert all(torch.equal(t, opt.flat_state()[k]) for k, t in held.items())
    # the tensor that it was made for, or another one like it, steps
    p.data = was.clone()
    p.grad = torch.ones_like(p)
    opt.step()
    assert not torch.equal(p.detach(), was)


def test_sizes_of_one_have_no_order(device):
    """Strides of dimensions of size 1 say nothing: converting such a tensor changes only them."""
    p = torch.nn.Parameter(torch.zeros(4, 3, 1, 1, device=device))
    opt = cx.AdamW([p], lr=0.1)
    p.data = p.data.as_strided(p.size(), (3, 1, 3, 3))
    p.grad = torch.ones_like(p)
    opt.step()
    assert (p.detach() < 0).all()


@pytest.mark.gpu
def test_a_module_that_moved_is_refused():
    for there, back in (("cpu", "cuda"), ("cuda", "cpu")):
        m = torch.nn.Linear(8, 8).to(there)
        opt = cx.AdamW(m.parameters(), lr=0.1)
        m.to(back)
        for p in m.parameters():
            p.grad = torch.ones_like(p)
        with pytest.raises(ComprexError, match="as it was"):
            opt.step()


def test_rounding_goes_on_while_another_tensor_rests(device):
    """A tensor with more steps that gets no gradient any more: the others' random bits are new ones at every step all the same, so
    their moments follow (bounds as in the test of one tensor)."""
    n = 4096
    p, rests = (torch.nn.Parameter(torch.zeros(n, device=device)) for _ in range(2))
    opt = cx.AdamW([p, rests], state_bits=8, lr=0.0, betas=(0.9, 0.98), weight_decay=0.0)
    rests.grad = torch.ones(n, device=device)
    for _ in range(200):
        opt.step()
    rests.grad = None
    p.grad = torch.ones(n, device=device)
    opt.step()
    p.grad = torch.full((n,), 0.25, device=device)
    p.grad[::256] = 1.0
    steps = 60
    for _ in range(steps):
        opt.step()
    keep = torch.arange(n) % 256 != 0
    got = (_decoded(opt, "exp_avg_rms")[0][keep] ** 2).mean().item()
    exact = 0.02 * 0.98 ** steps + 0.0625 * (1 - 0.98 ** steps)
    assert exact * 0.98 <= got <= exact * (1 + steps * 2.0 ** -8 * 1.05)
    # the first moment is near 0.25, in steps of 2^-5 of it at most 2^-3 wide; independent roundings, forgotten with 0.9 a step, have a
    # standard deviation below half a step / sqrt(1 - 0.81) each; their mean over n elements within five of its own
    exact = 0.1 * 0.9 ** steps + 0.25 * (1 - 0.9 ** steps)
    assert abs(_decoded(opt, "exp_avg")[0][keep].mean().item() - exact) <= 5 * (0.25 / 8 / 2 / (1 - 0.81) ** 0.5) / keep.sum().item() ** 0.5 + 0.25 * steps * 2.0 ** -16


def test_a_checkpoint_keeps_the_rounding(device):
    """The steps that make the random bits are the optimizer's own, whichever tensors took them."""
    def make():
        params = _params(torch.bfloat16, device, [700, 300])
        return params, cx.AdamW(params, state_bits=8, seed=1, **HYPER)

    def run(opt, params, steps):
        for t in steps:
            _set_grads(params, seed=t)
            params[t % 2].grad = None
            opt.step()
    a, whole = make()
    run(whole, a, range(6))
    b, part = make()
    run(part, b, range(3))
    c, other = make()
    other.load_state_dict(part.state_dict())
    run(other, c, range(3, 6))
    assert all(torch.equal(x, y) for x, y in zip(a, c))
    for k, t in whole.flat_state().items():
        assert torch.equal(t.view(torch.uint8), other.flat_state()[k].view(torch.uint8)), k
    # a file without the number of steps: that of the tensor with the most
    old = part.state_dict()
    del old["comprex_adamw"]["turns"]
    other.load_state_dict(old)


def test_a_graph_from_before_the_step_is_refused(device):
    """A step changes tensors in place, as autograd must know: a graph that still holds them cannot be gone back through."""
    w, b = (torch.nn.Parameter(torch.ones(*s, device=device)) for s in ((3, 5), (3,)))
    opt = cx.AdamW([w, b], lr=0.1)
    x = torch.ones(2, 5, device=device, requires_grad=True)
    y = cx.linear(x, w, b).square().sum()
    y.backward(retain_graph=True)
    b.grad = None
    versions = w._version, b._version
    opt.step()
    assert w._version > versions[0] and b._version == versions[1]       # only what has stepped
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    opt.zero_grad()
    cx.linear(x, w, b).sum().backward()                                 # a new graph is as good as any


def test_a_step_that_failed_does_not_count(device, monkeypatch):
    """Neither the tensors' step counts nor the optimizer's own move before the launch is out."""
    from comprex_b200 import _lib
    lib = _lib.load()

    class Failing:
        def __getattr__(self, name):
            return (lambda *a: -1) if name == "cx_adamw_step" else getattr(lib, name)
    params = _params(torch.bfloat16, device, [300, 5, 700])
    twin = _params(torch.bfloat16, device, [300, 5, 700])
    opt, clean = (cx.AdamW(x, state_bits=8, **HYPER) for x in (params, twin))
    for turn, missing in enumerate([(), (1,), (), (0, 2), ()]):
        for x in (params, twin):
            _set_grads(x, seed=turn)
            for i in missing:
                x[i].grad = None
        with monkeypatch.context() as m:
            m.setattr(_lib, "load", lambda: Failing())
            for _ in range(2):
                with pytest.raises(ComprexError):
                    opt.step()
        opt.step()
        clean.step()
    assert all(torch.equal(a, b) for a, b in zip(params, twin))
    for k, t in clean.flat_state().items():
        assert torch.equal(t.view(torch.uint8), opt.flat_state()[k].view(torch.uint8)), k
    assert opt.state_dict()["comprex_adamw"]["steps"] == clean.state_dict()["comprex_adamw"]["steps"] == [4, 4, 4]


def test_a_table_that_was_not_brought_over_is_sent_again(device):
    """Addresses that the device has not got are not taken for known: it would go on with the old ones."""
    class Broken:
        def copy_(self, *args, **kwargs):
            raise RuntimeError("no memory")
    params = _params(torch.float32, device, [300, 5, 700])
    twin = _params(torch.float32, device, [300, 5, 700])
    opt, clean = (cx.AdamW(x, **HYPER) for x in (params, twin))
    held = []
    for turn, name in enumerate(["seg_param", "seg_grad", "seg_class"]):
        for x in (params, twin):
            _set_grads(x, seed=turn)
            if name == "seg_param":
                held.append(x[0].data)
                x[0].data = x[0].data.clone()
            if name == "seg_class":
                x[1].grad = None
        table, opt._lay[name] = opt._lay[name], Broken()
        with pytest.raises(RuntimeError, match="no memory"):
            opt.step()
        opt._lay[name] = table
        opt.step()
        clean.step()
        assert all(torch.equal(a, b) for a, b in zip(params, twin)), name


@pytest.mark.parametrize("bits", [8, 32])
def test_every_tensor_its_own_step_count(device, bits):
    """More step counts than fit into one launch, and tensors that rest: as each tensor would step alone."""
    k = 150
    params = _params(torch.bfloat16, device, [40 + 7 * i for i in range(k)])
    opt = cx.AdamW(params, state_bits=bits, seed=2, **HYPER)
    launches = []
    for turn in range(k + 2):
        _set_grads(params, seed=turn)
        for i, p in enumerate(params):
            if i > turn:                          # tensor i steps from turn i on; at last there are 150 counts
                p.grad = None
        if turn < k - 3:
            opt._steps[:turn + 1] += 1            # (quickly: as if they had stepped)
            opt._classes = None
            continue
        counts = opt._steps.copy()
        before = cx.launch_count()
        exact = []
        held = (_decoded(opt, "exp_avg"), [r * r for r in _decoded(opt, "exp_avg_rms")]) if bits == 8 else \
            tuple([opt.flat_state()[s][a:a + n].double().cpu() for a, n in opt.spans()] for s in ("exp_avg", "exp_avg_sq"))
        for i, (w, p) in enumerate(zip(_weights(opt, params), params)):
            exact.append(w if p.grad is None else _formula(w, held[0][i], held[1][i], p.grad.double().cpu(), int(counts[i]) + 1, **HYPER)[0])
        opt.step()
        launches.append(cx.launch_count() - before)
        for got, w in zip(_weights(opt, params), exact):
            assert (got - w).abs().max() <= EPS32 * (2 * w.abs().max() + 10 * HYPER["lr"] * 8) + 1e-7
    assert opt.state_dict()["comprex_adamw"]["steps"] == [k + 2 - i for i in range(k)]
    if device == "cuda":
        assert launches[-1] == 3                  # 64 rows of settings each


def test_settings_of_tensors_that_rest_take_no_row(device):
    params = _params(torch.float32, device, [20] * 100)
    opt = cx.AdamW(params, **HYPER)
    for i, p in enumerate(params):
        for q in params:
            q.grad = None
        p.grad = torch.ones_like(p)
        before = cx.launch_count()
        opt.step()
        assert device != "cuda" or cx.launch_count() - before == 1
    assert opt.state_dict()["comprex_adamw"]["steps"] == [1] * 100


def test_the_negative_bit(device):
    """A gradient whose sign is only noted is one with that sign; a tensor of that kind is not one to step."""
    p, q = (torch.nn.Parameter(torch.ones(300, device=device)) for _ in range(2))
    g = torch.linspace(-1, 1, 300, device=device)
    p.grad, q.grad = torch._neg_view(g), -g
    cx.AdamW([p], lr=0.1).step()
    cx.AdamW([q], lr=0.1).step()
    assert torch.equal(p, q)
    noted = torch._neg_view(torch.ones(300, device=device)).requires_grad_()
    with pytest.raises(ComprexError):
        cx.AdamW([noted])


def test_tensors_without_memory_are_refused(device):
    """Fake tensors have no memory to step, or to read a gradient from; a gradient of zeros that is not written down is one."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    real, mode = torch.nn.Parameter(torch.zeros(300, device=device)), FakeTensorMode()
    with mode:
        with pytest.raises(ComprexError):
            cx.AdamW([torch.nn.Parameter(torch.zeros(300, device=device))])
        with pytest.raises(ComprexError):
            cx.AdamW([real])
    opt = cx.AdamW([real], lr=0.1)
    with mode:
        real.grad = torch.ones(300, device=device)
    with pytest.raises(ComprexError):
        opt.step()
    assert not real.detach().any()
    real.grad = None
    real.grad = torch._efficientzerotensor((300,), device=device)
    opt.step()
    assert not real.detach().any() and opt.state_dict()["comprex_adamw"]["steps"] == [1]


@pytest.mark.parametrize("bits", [8, 32])
def test_a_checkpoint_of_another_order_is_refused(device, bits):
    """The flat states are in the tensors' memory order: read in another one they would belong to other elements."""
    def make(order):
        p = torch.nn.Parameter(torch.randn(4, 3, 2, 2, generator=torch.Generator().manual_seed(0)).to(device, torch.bfloat16))
        p.data = order(p.data)
        opt = cx.AdamW([p], lr=0.1, state_bits=bits)
        p.grad = torch.ones_like(p)
        opt.step()
        return p, opt
    orders = [lambda t: t, lambda t: t.contiguous(memory_format=torch.channels_last), lambda t: t.reshape(3, 4, 2, 2), lambda t: t.reshape(12, 4)]
    for i, there in enumerate(orders):
        p, opt = make(there)
        before = p.detach().clone()
        for j, here in enumerate(orders):
            saved = make(here)[1].state_dict()
            if i == j:
                opt.load_state_dict(saved)
                continue
            with pytest.raises(ComprexError, match="order"):
                opt.load_state_dict(saved)
            assert torch.equal(p.detach(), before)
        # a file that does not say: taken to be in the tensors' order, as it was
        del saved["comprex_adamw"]["shapes"]
        opt.load_state_dict(saved)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_tensor_unfrozen_later_steps(device, dtype, bits):
    """Frozen when the optimizer is made, stepped from its first gradient on; the others go on as if nothing had happened."""
    sizes = [300, 5, 700, 1000]
    params = _params(dtype, device, sizes)
    for i in (0, 2):
        params[i].requires_grad_(False)
    opt = cx.AdamW([{"params": params[:2], "lr": 0.02}, {"params": params[2:]}], state_bits=bits, **HYPER)
    assert len(opt.spans()) == 2
    held = opt.flat_state()
    hyper = [HYPER | {"lr": 0.02}] * 2 + [HYPER] * 2
    saved = None
    for turn in range(6):
        live = [i for i in range(4) if i in (1, 3) or (i == 2 and turn >= 2) or (i == 0 and turn >= 4)]
        grads = [(torch.randn(n, generator=torch.Generator().manual_seed(10 * turn + i)) * 1e-2).to(dtype).to(device) for i, n in enumerate(sizes)]
        for i, p in enumerate(params):
            p.requires_grad_(i in live)
            p.grad = grads[i].clone() if i in live else None
        index = {id(p): j for j, p in enumerate(opt._params)}
        names = ("exp_avg", "exp_avg_rms") if bits == 8 else ("exp_avg", "exp_avg_sq")
        was = [_decoded(opt, n) if bits == 8 else [opt.flat_state()[n][a:a + k].double().cpu() for a, k in opt.spans()] for n in names]
        weights = _weights(opt, opt._params)
        want, count = {}, opt.state_dict()["comprex_adamw"]["steps"]
        for i in live:
            j = index.get(id(params[i]))
            zero = torch.zeros(sizes[i], dtype=torch.float64)
            w, m, v, t = (params[i].detach().double().cpu(), zero, zero, 0) if j is None else (weights[j], was[0][j], was[1][j], count[j])
            want[i] = _formula(w, m, v * v if bits == 8 else v, grads[i].double().cpu(), t + 1, **hyper[i])[0]
        frozen = {i: params[i].detach().clone() for i in range(4) if i not in live}
        opt.step()
        got = dict(zip((id(p) for p in opt._params), _weights(opt, opt._params)))
        for i, w in want.items():
            assert (got[id(params[i])] - w).abs().max() <= EPS32 * (2 * w.abs().max() + 10 * 0.02 * 8) + 1e-7, (turn, i)
        assert all(torch.equal(params[i].detach(), w) for i, w in frozen.items())
        assert len(opt.spans()) == (2 if turn < 2 else 3 if turn < 4 else 4)
        assert (opt.flat_state()["exp_avg"] is held["exp_avg"]) == (turn < 2)
        if turn == 2:
            saved = opt.state_dict(), [p.detach().clone() for p in params]
    assert opt.state_dict()["comprex_adamw"]["steps"] == [2, 6, 4, 6]
    # a checkpoint says which tensors it has
    fresh = [torch.nn.Parameter(w.clone(), requires_grad=i in (1, 3)) for i, w in enumerate(saved[1])]
    other = cx.AdamW([{"params": fresh[:2]}, {"params": fresh[2:]}], state_bits=bits)
    other.load_state_dict(saved[0])
    assert len(other.spans()) == 3 and other.state_dict()["comprex_adamw"]["steps"] == [3, 1, 3]
    opt.load_state_dict(saved[0])                 # and back, in the run that has gone on
    for k, t in saved[0]["comprex_adamw"]["flat"].items():
        assert torch.equal(t.view(torch.uint8), other.flat_state()[k].cpu().view(torch.uint8))
        assert torch.equal(t.view(torch.uint8), opt.flat_state()[k].cpu().view(torch.uint8))


def test_an_unfrozen_tensor_of_another_type_is_refused(device):
    p = torch.nn.Parameter(torch.ones(30, device=device))
    q = torch.nn.Parameter(torch.ones(30, device=device, dtype=torch.bfloat16), requires_grad=False)
    opt = cx.AdamW([p, q], lr=0.1)
    p.grad = torch.ones_like(p)
    opt.step()
    q.requires_grad_()
    q.grad = torch.ones_like(q)
    before = p.detach().clone()
    with pytest.raises(ComprexError):
        opt.step()
    assert torch.equal(p.detach(), before) and len(opt.spans()) == 1
    q.grad = None
    opt.step()
    assert opt.state_dict()["comprex_adamw"]["steps"] == [2]


@pytest.mark.parametrize("how", ["deepcopy", "pickle", "torch.save"])
@pytest.mark.parametrize("bits", [8, 32])
def test_copies_step_on(device, bits, how):
    """A copy, with the model or alone, goes on as the optimizer itself does, and neither disturbs the other."""
    import copy
    import io
    import pickle
    params = torch.nn.ParameterList(_params(torch.bfloat16, device, [300, 5, 700]))
    params.append(torch.nn.Parameter(torch.randn(4, 3, 2, 2).to(device, torch.bfloat16).contiguous(memory_format=torch.channels_last)))
    params[1].requires_grad_(False)
    opt = cx.AdamW(params, state_bits=bits, seed=4, **HYPER)

    def run(o, ps, turns):
        for t in turns:
            gen = torch.Generator().manual_seed(t)
            for i, p in enumerate(ps):
                g = (torch.randn(p.size(), generator=gen) * 1e-2).to(p.dtype).to(device)
                p.grad = None if i == 1 and t < 4 else torch.empty_like(p, requires_grad=False).copy_(g)
            o.step()
    run(opt, params, range(3))
    if how == "deepcopy":
        twins, other = copy.deepcopy((params, opt))
    elif how == "pickle":
        twins, other = pickle.loads(pickle.dumps((params, opt)))
    else:
        file = io.BytesIO()
        torch.save((params, opt), file)
        file.seek(0)
        twins, other = torch.load(file, weights_only=False)
    assert all(p is q for p, q in zip(other._params, [twins[0], twins[2], twins[3]]))
    before = [p.detach().clone() for p in params]
    run(other, twins, range(3, 6))
    assert all(torch.equal(p, q) for p, q in zip(params, before))
    run(opt, params, range(3, 6))
    assert all(torch.equal(p, q) for p, q in zip(params, twins))
    assert other.state_dict()["comprex_adamw"]["steps"] == [6, 2, 6, 6]
    for k, t in opt.flat_state().items():
        assert torch.equal(t.view(torch.uint8), other.flat_state()[k].view(torch.uint8)), k
