"""The operators together: GPT-2 with them, its example, and what they must bear in use (graphs, long offsets, memory)."""
import os
import subprocess
import sys

import pytest
import torch

import comprex_b200 as cx
from comprex_b200.models.gpt2 import gpt2_tiny

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _models(device, dtype=torch.float32):
    out = []
    for fused in (False, True):
        torch.manual_seed(0)
        out.append(gpt2_tiny(fused=fused).to(device, dtype))
    return out


def test_gpt2_with_and_without_the_operators(device):
    """In 32 bits both are the same sums in another order: a few hundred roundings of 2^-24 through two layers."""
    plain, fused = _models(device)
    idx = torch.randint(0, 257, (2, 33), generator=torch.Generator().manual_seed(1)).to(device)
    x, y = idx[:, :-1].contiguous(), idx[:, 1:].contiguous()
    losses = [m(x, y) for m in (plain, fused)]
    assert abs(losses[0].item() - losses[1].item()) <= 1e-5 * losses[0].item()
    grads = [torch.autograd.grad(loss, list(m.parameters())) for loss, m in zip(losses, (plain, fused))]
    for (name, _), a, b in zip(plain.named_parameters(), *grads):
        assert (a - b).norm() <= 1e-4 * a.norm() + 1e-9, name
    with torch.no_grad():
        a, b = plain(idx), fused(idx)
    assert (a - b).abs().max() <= 1e-5 * (1 + a.abs().max())


def test_a_step_of_everything_lowers_the_loss(device):
    _, model = _models(device, torch.bfloat16 if device == "cuda" else torch.float32)
    opt = cx.AdamW(model.parameters(), lr=3e-3, state_bits=8)
    start = torch.arange(0, 8)[:, None]
    seq = ((start + 3 * torch.arange(33)) % 257).to(device)
    first = None
    for _ in range(12):
        opt.zero_grad()
        loss = model(seq[:, :-1], seq[:, 1:])
        loss.backward()
        opt.step()
        first = loss.item() if first is None else first
    assert loss.item() < first - 1.0


def test_example_runs():
    env = dict(os.environ, CUDA_VISIBLE_DEVICES="", OMP_NUM_THREADS="2")
    res = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "gpt2_train.py"), "--steps", "10", "--generate", "2"], env=env, capture_output=True,
                         text=True, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr
    assert "mean loss over 1 ranks" in res.stdout and "generated" in res.stdout


@pytest.mark.gpu
def test_in_a_cuda_graph():
    gen = torch.Generator(device="cuda").manual_seed(0)
    make = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()  # noqa: E731
    x, w, b, v = make(200, 64), make(128, 64), make(128), make(1000, 128)
    t = torch.randint(0, 1000, (200,), generator=gen, device="cuda")
    one = make(1, 64)

    def call():
        h = cx.linear(x, w, b, activation="gelu_tanh")
        return h, cx.linear_cross_entropy(h, v, t), cx.linear(one, w, b)

    with torch.no_grad():
        want = [o.clone() for o in call()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        for o in got:
            o.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        x.copy_(make(200, 64))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, call()))


@pytest.mark.gpu
def test_results_of_more_than_2_31_elements():
    """The last rows of a result whose offsets pass 32 bits, aligned and not."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    for outer in (32768, 32771):
        rows = 66000
        x = torch.randn(rows, 64, generator=gen, device="cuda").bfloat16()
        w = torch.randn(outer, 64, generator=gen, device="cuda").bfloat16()
        y = cx.linear(x, w)
        assert rows * outer > 1 << 31
        for part in (slice(0, 40), slice(rows - 40, rows)):
            want = x[part].double() @ w.double().T
            assert ((y[part].double() - want).abs() <= 2.0 ** -8 * want.abs() + 64 * 2.0 ** -23 * (x[part].double().abs() @ w.double().abs().T)).all()
        del y


@pytest.mark.gpu
def test_adamw_beyond_2_31_elements():
    n = (1 << 31) + 4099
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    p.grad[-5:] = -1.0
    opt = cx.AdamW([p], lr=0.5, weight_decay=0.0, state_bits=8)
    opt.step()
    # m / c1 over sqrt(v / c2) is one: every weight moves by lr
    assert (p[:1000] == -0.5).all() and (p[-4000:-5] == -0.5).all() and (p[-5:] == 0.5).all()
    moved = opt.flat_state()["exp_avg"].view(torch.uint8)
    assert moved[n - 1] != 0 and not moved[n:].any()


@pytest.mark.gpu
def test_the_loss_holds_no_logits():
    rows, vocab, dim = 4096, 50257, 256
    h = torch.randn(rows, dim, device="cuda").bfloat16().requires_grad_()
    w = (torch.randn(vocab, dim, device="cuda") * 0.05).bfloat16().requires_grad_()
    t = torch.randint(0, vocab, (rows,), device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    loss = cx.linear_cross_entropy(h, w, t)
    logits = rows * vocab * 2
    assert torch.cuda.max_memory_allocated() - before < logits / 10
    torch.autograd.grad(loss, (h, w))
    # a piece of the probabilities, sums and gradients
    assert torch.cuda.max_memory_allocated() - before < (288 << 20) + 2 * (rows + vocab) * dim * 2 + 4 * rows * dim + (1 << 20)


@pytest.mark.gpu
def test_operands_of_another_stream():
    gen = torch.Generator(device="cuda").manual_seed(3)
    h = torch.randn(300, 128, generator=gen, device="cuda").half()
    w = torch.randn(2000, 128, generator=gen, device="cuda").half() * 0.1
    t = torch.randint(0, 2000, (300,), generator=gen, device="cuda")
    a, b = (x.clone().requires_grad_() for x in (h, w))
    want = [x.clone() for x in torch.autograd.grad(cx.linear_cross_entropy(a, b, t), (a, b))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.autograd.grad(cx.linear_cross_entropy(a, b, t), (a, b))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_gpt2_under_autocast(device):
    """The model with and without the operators, weights in 32 bits: the same types, and the same numbers but for bf16 roundings."""
    plain, fused = _models(device)
    idx = torch.randint(0, 257, (2, 33), generator=torch.Generator().manual_seed(1)).to(device)
    losses, logits = [], []
    for m in (plain, fused):
        with torch.autocast(device, dtype=torch.bfloat16):
            losses.append(m(idx[:, :-1], idx[:, 1:].contiguous()))
            logits.append(m(idx))
        losses[-1].backward()
    assert losses[0].dtype == losses[1].dtype and logits[0].dtype == logits[1].dtype
    # logits of a tiny model near zero: rounded to 2^-9 of themselves in both, and so are the activations before them
    assert abs(losses[0].item() - losses[1].item()) <= 2.0 ** -8 * losses[0].item()
    assert (logits[0] - logits[1]).norm() <= 2.0 ** -5 * logits[0].norm()
    for (name, p), q in zip(plain.named_parameters(), fused.parameters()):
        assert q.grad.dtype == torch.float32 and (p.grad - q.grad).norm() <= 2.0 ** -4 * p.grad.norm() + 1e-6, name


FIRST_IN_A_GRAPH = """
import torch
import comprex_b200 as cx
torch.manual_seed(0)
x, w, v = (torch.randn(*s, device="cuda").bfloat16() for s in ((200, 64), (128, 64), (1000, 128)))
t = torch.randint(0, 1000, (200,), device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.no_grad(), torch.cuda.graph(graph):
    h = cx.linear(x, w)
    loss = cx.linear_cross_entropy(h, v, t)
graph.replay()
got = h.clone(), loss.clone()
with torch.no_grad():
    h = cx.linear(x, w)
    loss = cx.linear_cross_entropy(h, v, t)
assert torch.equal(got[0], h) and torch.equal(got[1], loss) and torch.isfinite(loss)
print("the same")
"""


@pytest.mark.gpu
def test_the_first_product_of_a_process_in_a_cuda_graph():
    """What a process sets up once is set up under a capture, too."""
    res = subprocess.run([sys.executable, "-c", FIRST_IN_A_GRAPH], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "the same" in res.stdout, res.stdout + res.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["pairs", "rle", "dense"])
@pytest.mark.parametrize("rows", [1, 64, 1024])
def test_operators_between_send_and_receive(kind, rows):
    """The receiver's vector is what a product of this package has just written (its kernels let the kernel behind in early): small
    whole numbers, so everything is exact."""
    cols = 1024
    n = rows * cols
    dtype = torch.bfloat16 if kind != "rle" else torch.float32
    env = cx.GaspiEnvironment(8 << 20, device="cuda")
    ex = cx.GaspiEx(env, n, dtype=dtype) if kind == "dense" else cx.Comprex(env, n)
    if kind != "dense":
        ex.setThreshold(cx.ThresholdTopK(0.05))
        ex.setCompressor(cx.CompressorRLE() if kind == "rle" else cx.CompressorIndexPairs())
    ex.connectTo(0, 0)
    gen = torch.Generator(device="cuda").manual_seed(rows)
    held = torch.zeros(n, device="cuda")
    for _ in range(8):
        v = torch.randint(-9, 10, (n,), device="cuda", generator=gen).to(dtype)
        x, w = (torch.randint(-2, 3, (k, 32), device="cuda", generator=gen).to(torch.bfloat16) for k in (rows, cols))
        want = x.float() @ w.float().T
        ex.writeRemote(v)
        out = cx.linear(x, w).view(n)
        out = out if kind != "rle" else out.float()
        ex.readRemote_add(out)
        held += v.float()
        sent = v.float()
        if kind != "dense":
            sent, held = held - ex.getRests(), ex.getRests()
        assert torch.equal(out.float(), want.view(n) + sent)
    env.check()
    env.close()
