"""Times that stand beside the operators of a training step, on one GPU: GPT-2 medium's step with and without them, single
products beside the library's, AdamW on one large tensor, and its step when the gradients' addresses change.

    python bench/operators_bench.py --out results/operators.txt

Device time with CUDA events after warm-up.  Single products go round copies of their operands that together are larger than L2;
``burst`` is a short run after a pause, ``sustained`` one of two seconds, at the power limit.  The median SM clock under load and the
throttle reasons seen are printed with each part.
"""
import argparse
import os
import statistics
import subprocess
import sys
import time

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

import comprex_b200 as cx  # noqa: E402
from comprex_b200.models.gpt2 import gpt2_medium  # noqa: E402


class Clocks:
    """SM clock and throttle reasons while the body runs."""

    def __enter__(self):
        self.p = subprocess.Popen(["nvidia-smi", "--query-gpu=clocks.sm,utilization.gpu,clocks_event_reasons.active", "--format=csv,noheader,nounits",
                                   "-lms", "100"], stdout=subprocess.PIPE, text=True)
        return self

    def __exit__(self, *exc):
        self.p.terminate()
        rows = [line.split(", ") for line in self.p.communicate()[0].splitlines()]
        busy = [r for r in rows if len(r) == 3 and r[1].isdigit() and int(r[1]) > 0] or rows
        self.text = f"SM {statistics.median(int(r[0]) for r in busy):.0f} MHz, reasons {sorted({r[2] for r in busy})}" if busy else "no samples"


def timed(f, n):
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    a.record()
    for i in range(n):
        f(i)
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b) / n * 1e3


def product(rows, inner, outer, say):
    sets = max(2, (300 << 20) // (2 * (rows * inner + inner * outer)))
    sets = min(sets, 64)
    xs, ws = ([torch.randn(*s, device="cuda").bfloat16() for _ in range(sets)] for s in ((rows, inner), (outer, inner)))
    calls = {"linear": lambda i: cx.linear(xs[i % sets], ws[i % sets]), "library": lambda i: torch.nn.functional.linear(xs[i % sets], ws[i % sets])}
    out = {}
    with torch.no_grad():
        for name, f in calls.items():
            timed(f, 3)
            time.sleep(0.5)
            burst = min(timed(f, 10) for _ in range(3))
            out[name] = burst, timed(f, max(10, int(2e6 / burst)))
    say(f"{rows} x {inner} -> {outer}: " + ", ".join(f"{k} {b:.1f} us burst, {s:.1f} sustained" for k, (b, s) in out.items()))


def gpt2(fused, which, say):
    torch.manual_seed(0)
    model = gpt2_medium(fused=fused).cuda().bfloat16()
    opt = (torch.optim.AdamW(model.parameters(), lr=1e-4, fused=True) if which == "torch"
           else cx.AdamW(model.parameters(), lr=1e-4, state_bits=int(which)))
    x, y = (torch.randint(0, 50257, (8, 1024), device="cuda") for _ in range(2))

    def step(_):
        opt.zero_grad()
        model(x, y).backward()
        opt.step()
    torch.cuda.reset_peak_memory_stats()
    timed(step, 5)
    with Clocks() as c:
        t = timed(step, 40)
    say(f"fused={fused}, AdamW {which}: {t / 1e3:.2f} ms a step, {torch.cuda.max_memory_allocated() / 1e9:.1f} GB; {c.text}")


def adamw(dtype, bits, say, n=256 << 20):
    p = torch.nn.Parameter((torch.randn(n, device="cuda") * 0.02).to(dtype))
    p.grad = (torch.randn(n, device="cuda") * 1e-3).to(dtype)
    opt = cx.AdamW([p], state_bits=bits)
    timed(lambda i: opt.step(), 5)
    t = timed(lambda i: opt.step(), 50)
    per = {torch.float32: 12, torch.bfloat16: 12}[dtype] + (16 if bits == 32 else 4)      # gradient, weights both ways (and copy), states both ways
    say(f"{n} elements, {dtype}, states of {bits} bits: {t:.0f} us, {n * per / t / 1e6:.2f} TB/s")


def host_side(count, say):
    """Host time of a step: gradients where they were, at new addresses each time, and the first step."""
    params = [torch.nn.Parameter(torch.zeros(256, device="cuda")) for _ in range(count)]
    t0 = time.perf_counter()
    opt = cx.AdamW(params)
    torch.cuda.synchronize()
    made = time.perf_counter() - t0
    grads = [[torch.zeros(256, device="cuda") for _ in params] for _ in range(2)]

    def step(which):
        for p, g in zip(params, grads[which]):
            p.grad = g
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        opt.step()
        torch.cuda.synchronize()
        return (time.perf_counter() - t0) * 1e6
    first = step(0)
    same = statistics.median(step(0) for _ in range(50))
    moved = statistics.median(step(i % 2) for i in range(50))
    say(f"{count} tensors: made in {made * 1e6:.0f} us, first step {first:.0f}, then {same:.0f}, with gradients at new addresses {moved:.0f} (host and GPU, waited for)")


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--out")
    args = ap.parse_args()
    lines = []

    def say(text):
        print(text, flush=True)
        lines.append(text)
    host_side(10, lambda text: None)              # (the process's own start)
    for count in (10, 161, 292):
        host_side(count, say)
    for dtype in (torch.bfloat16, torch.float32):
        for bits in (32, 8):
            with Clocks() as c:
                adamw(dtype, bits, say)
            say("  " + c.text)
    for size in ((1024, 1024, 1024), (8192, 1024, 4096), (8192, 4096, 1024), (8192, 4096, 4096), (8192, 8192, 8192)):
        with Clocks() as c:
            product(*size, say)
        say("  " + c.text)
    for rows in (1, 2, 3, 4, 8, 16):
        for size in ((1024, 4096), (4096, 1024), (4096, 4096)):
            product(rows, *size, say)
    for fused, which in ((False, "torch"), (True, "torch"), (True, "32"), (True, "8")):
        gpt2(fused, which, say)
        torch.cuda.empty_cache()
    if args.out:
        with open(args.out, "w") as f:
            f.write("\n".join(lines) + "\n")


if __name__ == "__main__":
    main()
