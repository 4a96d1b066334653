"""The loss over a vocabulary without its logits (csrc/vocab_loss.cu) and its gradients, against 64 bits."""
import math

import pytest
import torch

import comprex_b200 as cx
from comprex_b200 import ComprexError

TYPES = [torch.float32, torch.bfloat16, torch.float16]
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # unit roundoff: 24, 8 and 11 bits
SMALL = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}                 # half a subnormal step
# rows, vocabulary, width: one of everything, tile borders, odd sizes
SIZES = [(1, 257, 64), (1, 1, 8), (3, 2, 5), (64, 256, 64), (65, 513, 72), (130, 1000, 33), (300, 255, 96), (257, 130, 264)]


def _inputs(rows, vocab, dim, dtype, device, ignored=0.2, spread=2.0, seed=0):
    gen = torch.Generator().manual_seed(seed)
    h = torch.randn(rows, dim, generator=gen).to(dtype).to(device)
    w = (torch.randn(vocab, dim, generator=gen) * spread / dim ** 0.5).to(dtype).to(device)
    t = torch.randint(0, vocab, (rows,), generator=gen)
    t[torch.rand(rows, generator=gen) < ignored] = -100
    t[0] = vocab - 1
    return h, w, t.to(device), (torch.rand(rows, generator=gen) + 0.5).to(device)


def _check(h, w, t, g, reduction, loss, dh, dw):
    """Elementwise bounds: logits off by n 2^-23 times their sum of magnitudes, losses by twice that and a few roundings;
    the probabilities by as much, and by their rounding to the type (times 2^13 / the largest factor, for fp16)."""
    unit, small = UNIT[h.dtype], SMALL[h.dtype]
    H, W, T, G = h.double().cpu(), w.double().cpu(), t.cpu(), g.double().cpu()
    rows, dim = H.shape
    kept = (T != -100).double()
    s = H @ W.T
    lse = torch.logsumexp(s, 1)
    hot = torch.zeros_like(s).scatter_(1, T.clamp_min(0)[:, None], 1.0)
    each = (lse - (s * hot).sum(1)) * kept
    e_s = ((dim + 4) * 2.0 ** -23 * (H.abs() @ W.abs().T)).amax(1)
    e_loss = 2 * e_s + 2.0 ** -21 * (1 + s.abs().amax(1) + lse.abs())
    n = kept.sum()
    if reduction == "none":
        want, e_want = each, e_loss
    else:
        want, e_want = each.sum(), e_loss.sum() + 2.0 ** -23 * rows * each.abs().sum() * 0.1 + 2.0 ** -22 * each.sum()
        if reduction == "mean":
            want, e_want = want / n, e_want / n
    assert loss.dtype == torch.float32
    assert ((loss.detach().double().cpu() - want).abs() <= e_want).all()
    if dh is None:
        return
    f = G * kept if reduction == "none" else G * kept / (n if reduction == "mean" else 1.0)
    prob = torch.exp(s - lse[:, None])
    p = (prob - hot) * f[:, None]
    e_p = prob * f.abs()[:, None] * (2 * e_loss[:, None] + 2.0 ** -20) + unit * p.abs() * 1.01 + small * 2.0 ** -12 * f.abs().max()
    for got, want, bound in ((dh, p @ W, e_p @ W.abs() + (W.size(0) + 8) * 2.0 ** -23 * (p.abs() @ W.abs())),
                             (dw, p.T @ H, e_p.T @ H.abs() + (rows + 8) * 2.0 ** -23 * (p.abs().T @ H.abs()))):
        if got is not None:
            assert ((got.double().cpu() - want).abs() <= 1.01 * (bound + unit * want.abs() + small)).all()


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_against_64_bits(device, dtype, size, reduction):
    h, w, t, g = _inputs(*size, dtype, device)
    if reduction != "none":
        g = g[0]
    h.requires_grad_(), w.requires_grad_()
    loss = cx.linear_cross_entropy(h, w, t, reduction=reduction)
    dh, dw = torch.autograd.grad(loss, (h, w), g)
    _check(h.detach(), w.detach(), t, g, reduction, loss, dh, dw)
    assert not dh[t == -100].any()
    with torch.no_grad():
        assert torch.equal(cx.linear_cross_entropy(h, w, t, reduction=reduction), loss)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(1, 50257, 1024), (7, 50257, 136), (2000, 1003, 64), (1025, 5000, 1000), (128, 40000, 8), (4500, 20000, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_larger_sizes(size, dtype):
    """Among them several pieces of the vocabulary."""
    h, w, t, g = _inputs(*size, dtype, "cuda")
    h.requires_grad_(), w.requires_grad_()
    loss = cx.linear_cross_entropy(h, w, t, reduction="none")
    dh, dw = torch.autograd.grad(loss, (h, w), g)
    _check(h.detach(), w.detach(), t, g, "none", loss, dh, dw)
    again = cx.linear_cross_entropy(h, w, t, reduction="none")
    assert torch.equal(loss, again) and all(torch.equal(a, b) for a, b in zip((dh, dw), torch.autograd.grad(again, (h, w), g)))


def test_one_gradient_only(device):
    h, w, t, g = _inputs(70, 300, 40, torch.bfloat16, device)
    both = [x.clone().requires_grad_() for x in (h, w)]
    want = torch.autograd.grad(cx.linear_cross_entropy(*both, t), both)
    for i in range(2):
        part = [x.clone().requires_grad_(i == j) for j, x in enumerate((h, w))]
        got, = torch.autograd.grad(cx.linear_cross_entropy(*part, t), [part[i]])
        assert torch.equal(got, want[i])


def test_memory_orders(device):
    gen = torch.Generator().manual_seed(0)
    wide_h, wide_w = torch.randn(6, 10, 90, generator=gen).bfloat16().to(device), torch.randn(400, 70, generator=gen).bfloat16().to(device)
    t = torch.randint(0, 200, (10, 6), generator=gen).to(device).T
    h, w = wide_h[:, :, 8:72], wide_w[::2, 3:67]
    loss = cx.linear_cross_entropy(h, w, t, reduction="none")
    assert loss.shape == (6, 10)
    flat = cx.linear_cross_entropy(h.reshape(60, 64).contiguous(), w.contiguous(), t.reshape(60), reduction="none")
    assert torch.equal(loss.view(60), flat)
    # an expanded gradient, and one of several dimensions
    a, b = h.detach().requires_grad_(), w.detach().requires_grad_()
    ones = torch.autograd.grad(cx.linear_cross_entropy(a, b, t, reduction="none").sum(), (a, b))
    full = torch.autograd.grad(cx.linear_cross_entropy(a, b, t, reduction="sum"), (a, b))
    assert all(torch.equal(x, y) for x, y in zip(ones, full))


def test_rows_that_do_not_count(device):
    h, w, t, _ = _inputs(20, 100, 16, torch.bfloat16, device, ignored=0.0)
    h.requires_grad_(), w.requires_grad_()
    none = torch.full_like(t, -100)
    loss = cx.linear_cross_entropy(h, w, none)
    assert torch.isnan(loss)
    assert all(not x.any() for x in torch.autograd.grad(loss, (h, w)))
    assert cx.linear_cross_entropy(h, w, none, reduction="sum").item() == 0.0
    # another number that is ignored, one that is a word of the vocabulary
    some = t.clone()
    some[3:9] = 7
    a = cx.linear_cross_entropy(h, w, some, ignore_index=7)
    b = cx.linear_cross_entropy(h, w, torch.where(some == 7, -100, some))
    assert torch.equal(a, b)
    # no rows at all
    assert torch.isnan(cx.linear_cross_entropy(h[:0], w, t[:0])) and cx.linear_cross_entropy(h[:0], w, t[:0], reduction="sum").item() == 0.0
    dw, = torch.autograd.grad(cx.linear_cross_entropy(h[:0], w, t[:0], reduction="sum"), (w,))
    assert not dw.any()


def test_a_target_outside_the_vocabulary(device):
    h, w, t, g = _inputs(20, 100, 16, torch.bfloat16, device, ignored=0.0)
    h.requires_grad_()
    for wrong in (100, -1, 1 << 40):
        bad = t.clone()
        bad[5] = wrong
        loss = cx.linear_cross_entropy(h, w, bad, reduction="none")
        assert torch.isnan(loss).nonzero().flatten().tolist() == [5]
        dh, = torch.autograd.grad(loss, (h,), g)
        assert torch.isnan(dh[5]).all() and torch.isfinite(dh[torch.arange(20, device=device) != 5]).all()


def test_special_values(device):
    """A logit of -inf is a word that cannot come; large logits do not overflow; a row that is no number stays one row."""
    h, w, t, _ = _inputs(20, 300, 16, torch.float32, device, ignored=0.0)
    h[:, 0], w[:, 0] = 1.0, 0.0
    low = w.clone()
    low[37:295, 0] = float("-inf")
    t = t % 37
    got = cx.linear_cross_entropy(h, low, t, reduction="none")
    want = cx.linear_cross_entropy(h, torch.cat((w[:37], w[295:])), t, reduction="none")
    assert torch.isfinite(got).all() and (got - want).abs().max() <= 1e-5
    big = cx.linear_cross_entropy(h * 1000, w, t, reduction="none")
    exact = torch.nn.functional.cross_entropy((h * 1000).double() @ w.double().T, t, reduction="none")
    assert ((big - exact).abs() <= 2.0 ** -20 * 4000 * 4).all()
    bad = h.clone()
    bad[4, 3] = float("nan")
    loss = cx.linear_cross_entropy(bad, w, t, reduction="none")
    assert torch.isnan(loss).nonzero().flatten().tolist() == [4]


def test_small_gradients_of_half_precision(device):
    """A mean over many rows: factors far below what fp16 holds reach the gradients all the same."""
    h, w, t, _ = _inputs(64, 200, 32, torch.float16, device, ignored=0.0)
    h.requires_grad_()
    g = torch.full((64,), 2.0 ** -40, device=device)
    g[0] = 2.0 ** -38
    dh, = torch.autograd.grad(cx.linear_cross_entropy(h, w, t, reduction="none") * 1.0, (h,), g * 2.0 ** 35)
    p = torch.softmax(h.detach().double().cpu() @ w.double().cpu().T, 1)
    p[torch.arange(64), t.cpu()] -= 1
    want = (p @ w.double().cpu()) * (g * 2.0 ** 35).double().cpu()[:, None]
    # the probabilities' rounding, and the result's, which is subnormal here
    assert ((dh.double().cpu() - want).abs() <= 2.0 ** -10 * (p.abs() @ w.double().cpu().abs()) * g.max().item() * 2.0 ** 35 + 2.0 ** -24).all()


def test_gradient_against_differences(device):
    h, w, t, _ = _inputs(12, 50, 10, torch.float32, device)
    h.requires_grad_(), w.requires_grad_()
    grads = torch.autograd.grad(cx.linear_cross_entropy(h, w, t, reduction="sum"), (h, w))
    for i, grad in enumerate(grads):
        way, step = torch.randn_like(grad), 1e-2
        moved = [[x + s * step * way if i == j else x for j, x in enumerate((h, w))] for s in (1, -1)]
        with torch.no_grad():
            high, low = (cx.linear_cross_entropy(*m, t, reduction="none").double().sum().item() for m in moved)
        # third derivatives of a loss are below the cube of the logits' change; the losses' own error over the step
        change = (moved[0][0].detach() @ moved[0][1].detach().T - moved[1][0].detach() @ moved[1][1].detach().T).abs().max().item() / 2 / step
        assert abs((grad.double() * way.double()).sum().item() - (high - low) / 2 / step) <= 12 * (step ** 2 * change ** 3 + 2.0 ** -20 * 8 / step)


def test_uniform_logits(device):
    h, w = torch.zeros(9, 24, device=device), torch.randn(1000, 24, device=device)
    loss = cx.linear_cross_entropy(h, w, torch.arange(9, device=device))
    assert abs(loss.item() - math.log(1000)) <= 1e-5


def test_refusals(device):
    h, w, t, _ = _inputs(8, 30, 16, torch.bfloat16, device)
    with pytest.raises(ValueError):
        cx.linear_cross_entropy(h, w, t, reduction="max")
    for bad in (dict(weight=w.float()), dict(hidden=h[:, :4]), dict(targets=t[:3]), dict(targets=t.int()), dict(targets=t.tolist()),
                dict(weight=w[0]), dict(hidden=h.double(), weight=w.double())):
        with pytest.raises(ComprexError):
            cx.linear_cross_entropy(**(dict(hidden=h, weight=w, targets=t) | bad))


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_the_negative_bit(device, reduction, which):
    """A tensor whose sign is only noted counts with its sign, the gradient that comes in, too."""
    h, w, t, g = _inputs(20, 90, 16, torch.bfloat16, device)
    if reduction != "none":
        g = g[0]
    got = []
    for s in (torch.neg, torch._neg_view):
        leaves = [(s(x.clone()) if i == which else x.clone()).detach().requires_grad_() for i, x in enumerate((h, w))]
        loss = cx.linear_cross_entropy(*leaves, t, reduction=reduction)
        got.append([loss, *torch.autograd.grad(loss, leaves, s(g) if which == 2 else g)])
    assert all(torch.equal(p.resolve_neg(), q.resolve_neg()) for p, q in zip(*got))


def test_forward_mode_is_refused(device):
    """A tangent is not dropped in silence: there is no forward-mode derivative."""
    h, w, t, g = _inputs(8, 30, 16, torch.float32, device)
    with torch.autograd.forward_ad.dual_level():
        for i in range(2):
            args = [torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)) if i == j else x for j, x in enumerate((h, w))]
            with pytest.raises(ComprexError, match="forward-mode"):
                cx.linear_cross_entropy(*args, t)
        leaf = h.clone().requires_grad_()
        up = torch.autograd.forward_ad.make_dual(g, torch.ones_like(g))
        with pytest.raises(ComprexError, match="forward-mode"):
            torch.autograd.grad(cx.linear_cross_entropy(leaf, w, t, reduction="none"), leaf, up)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", TYPES)
def test_a_bad_gradient_stays_with_its_row(device, dtype, bad):
    """A row whose upstream gradient is no number does not change what the other rows are scaled by."""
    h, w, t, g = _inputs(40, 200, 32, dtype, device, ignored=0.0)
    h.requires_grad_()
    got = []
    for value in (0.0, bad):
        up = g.clone()
        up[7] = value
        got.append(torch.autograd.grad(cx.linear_cross_entropy(h, w, t, reduction="none"), (h,), up)[0])
    keep = torch.arange(40, device=device) != 7
    assert got[0][keep].abs().amin(1).min() > 0 and torch.equal(got[0][keep], got[1][keep])
    assert not got[0][7].any() and not torch.isfinite(got[1][7]).any()


@pytest.mark.parametrize("far", [8, 20, 30])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_far_apart(device, dtype, far):
    """Rows whose upstream gradients are up to 2^-30 of the largest.  In fp16 the probabilities share one power of two, so a small row's
    are off by up to 2^-25 of 2^-12 of the largest gradient each, as the elementwise bounds say; in the row's own measure that is nothing
    down to 2^-16 (there within three roundings of the result)."""
    h, w, t, g = _inputs(90, 700, 48, dtype, device, ignored=0.0)
    g = torch.exp2(-torch.arange(90, device=device) * (far / 89.0)) * (2.0 ** 12 if dtype == torch.float16 else 1.0)
    h.requires_grad_(), w.requires_grad_()
    loss = cx.linear_cross_entropy(h, w, t, reduction="none")
    dh, dw = torch.autograd.grad(loss, (h, w), g)
    _check(h.detach(), w.detach(), t, g, "none", loss, dh, dw)
    p = torch.softmax(h.detach().double() @ w.detach().double().T, 1)
    p[torch.arange(90), t] -= 1
    want = (p * g.double()[:, None]) @ w.detach().double()
    near = g >= 2.0 ** -16 * g[0]
    assert ((dh.double() - want).norm(dim=1) <= (3 * UNIT[dtype] + 2.0 ** -18) * want.norm(dim=1))[near].all()


def test_autocast(device):
    """The product is in autocast's type, as torch's; the loss in 32 bits as ever."""
    h, w, t, _ = _inputs(20, 90, 16, torch.float32, device)
    leaves, cast = [x.clone().requires_grad_() for x in (h, w)], [x.bfloat16().requires_grad_() for x in (h, w)]
    with torch.autocast(device, dtype=torch.bfloat16):
        loss = cx.linear_cross_entropy(*leaves, t)
    want = cx.linear_cross_entropy(*cast, t)
    assert loss.dtype == torch.float32 and torch.equal(loss, want)
    assert all(torch.equal(p, q.float()) for p, q in zip(torch.autograd.grad(loss, leaves), torch.autograd.grad(want, cast)))


def test_sizes_beyond_the_tiles_are_refused():
    """As many tiles as 32 bits count once round: an error of the call (in a process of its own), not of the arithmetic."""
    import os
    import subprocess
    import sys
    code = """
import ctypes as C
from comprex_b200 import _lib
lib, l = _lib.load(), _lib.VocabLoss()
l.rows, l.vocab, l.dim, l.ldh, l.ldw, l.dtype = 1 << 25, 1 << 23, 8, 8, 8, 1
for name in ("h", "w", "targets", "loss", "lse", "count", "grad", "dh", "dw"):
    setattr(l, name, 1 << 20)
for back in (0, 1):
    assert lib.cx_vocab_loss_workspace_bytes(1, C.byref(l), back) > 0
    print(lib.cx_last_error().decode())
"""
    assert code.count("l.dtype") == 1
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, "-c", code], cwd=root, env=dict(os.environ, CUDA_VISIBLE_DEVICES=""), capture_output=True, text=True, timeout=200)
    assert res.returncode == 0 and "too many tiles" in res.stdout, res


@pytest.mark.gpu
def test_many_words_in_32_bits():
    """More tiles of the vocabulary than a grid's second dimension has."""
    vocab = 64 * 65535 + 70
    h = torch.ones(3, 1, device="cuda", requires_grad=True)
    w = torch.zeros(vocab, 1, device="cuda", requires_grad=True)
    t = torch.tensor([0, vocab - 1, 77], device="cuda")
    loss = cx.linear_cross_entropy(h, w, t, reduction="none")
    # a sum of `vocab` equal terms over tiles: its roundings are below 2^-20 of it
    assert (loss - math.log(vocab)).abs().max() <= 2.0 ** -20 * (1 + math.log(vocab))
    dw, = torch.autograd.grad(loss.sum(), (w,))
    want = torch.full((vocab, 1), 3.0 / vocab, device="cuda", dtype=torch.float64)
    want[t] -= 1.0
    assert ((dw.double() - want).abs() <= 2.0 ** -18 * want.abs()).all()


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype,rows,off", [(torch.bfloat16, 4080, 2.0 ** -11), (torch.float16, 4094, 2.0 ** -14)])
def test_gradients_have_no_common_error(device, dtype, rows, off, reduction):
    """A gradient that all rows share, here one that lies half-way between two numbers of the type (1 / 255 and 1 / 2047 times a power of
    two), is not rounded with every probability: what is left are roundings of their own, up to UNIT / sqrt(3) in a row and averaged over the
    rows, five standard deviations of which are 5 * 2^-8 / 1.7 / 64 = 2^-12.4 in bf16 and 2^-15.4 in fp16."""
    h, w, t, _ = _inputs(rows, 257, 64, dtype, device, ignored=0.0)
    h.requires_grad_(), w.requires_grad_()
    loss = cx.linear_cross_entropy(h, w, t, reduction=reduction)
    up = torch.ones((), device=device) * 64.0 if reduction == "mean" else torch.full((rows,), 64.0 / rows, device=device)
    got = torch.autograd.grad(loss, (h, w), up)
    p = torch.softmax(h.detach().double() @ w.detach().double().T, 1)
    p[torch.arange(rows), t] -= 1
    p *= 64.0 / rows
    for g, want in zip(got, (p @ w.detach().double(), p.T @ h.detach().double())):
        assert abs((g.double() * want).sum().item() / want.square().sum().item() - 1) <= off


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(300, 1500, 130), (2700, 21000, 20)])
def test_larger_sizes_in_32_bits(size):
    """Many tiles, and several pieces of the vocabulary."""
    h, w, t, g = _inputs(*size, torch.float32, "cuda")
    h.requires_grad_(), w.requires_grad_()
    loss = cx.linear_cross_entropy(h, w, t, reduction="none")
    dh, dw = torch.autograd.grad(loss, (h, w), g)
    _check(h.detach(), w.detach(), t, g, "none", loss, dh, dw)
