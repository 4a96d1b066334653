"""GPT-2 with this package's operators from the batch to the weights, data parallel.

Products with bias, GELU and residual in their epilogues, a loss that never holds the logits, gradients averaged by the
compressed exchange of the communication hook, and AdamW with 8-bit states in one launch for all tensors.

    torchrun --nnodes=1 --nproc-per-node 2 --master-addr 127.0.0.1 examples/gpt2_train.py --steps 50
    python examples/gpt2_train.py --steps 50 --generate 16           # one process

``--model medium`` trains the 355 M configuration.  Runs on GPUs (one process per GPU; bfloat16) or on CPU ranks (float32).
"""
import argparse
import os
import sys

import torch
import torch.distributed as dist
from torch.nn.parallel import DistributedDataParallel as DDP

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import comprex_b200 as cx  # noqa: E402
from comprex_b200.ddp_hook import ComprexHookState, comprex_hook  # noqa: E402
from comprex_b200.models.gpt2 import gpt2_medium, gpt2_tiny  # noqa: E402


def batch(size, ctx, vocab, gen, dev):
    """Sequences that count on by a step of their own: what comes next can be learned."""
    start, step = (torch.randint(1, n, (size, 1), generator=gen) for n in (vocab, 4))
    seq = (start + step * torch.arange(ctx + 1)) % vocab
    return seq[:, :-1].to(dev), seq[:, 1:].to(dev)


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=50)
    ap.add_argument("--model", choices=["tiny", "medium"], default="tiny")
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--ratio", type=float, default=0.05)
    ap.add_argument("--lr", type=float, default=3e-3)
    ap.add_argument("--state-bits", type=int, choices=[8, 32], default=8)
    ap.add_argument("--generate", type=int, default=0, help="tokens to generate, one by one, after training")
    args = ap.parse_args()
    cx.initGaspiCxx()
    env = cx.GaspiEnvironment((64 if args.model == "tiny" else 6 << 10) << 20)
    rank, ranks, dev = env.get_rank(), env.get_ranks(), env.device
    torch.manual_seed(0)
    dtype = torch.bfloat16 if dev.type == "cuda" else torch.float32
    model = (gpt2_tiny if args.model == "tiny" else gpt2_medium)(fused=True).to(dev, dtype)
    vocab, ctx = model.wte.num_embeddings, model.wpe.num_embeddings
    net = model
    if ranks > 1:
        net = DDP(model, device_ids=[dev.index] if dev.type == "cuda" else None)
        net.register_comm_hook(ComprexHookState(env, compression_ratio=args.ratio), comprex_hook)
    # norms and biases are not decayed
    decay, plain = [], []
    for p in model.parameters():
        (decay if p.dim() > 1 else plain).append(p)
    opt = cx.AdamW([{"params": decay, "weight_decay": 0.1}, {"params": plain, "weight_decay": 0.0}], lr=args.lr, betas=(0.9, 0.95),
                   state_bits=args.state_bits)
    gen = torch.Generator().manual_seed(rank)
    for step in range(args.steps):
        x, y = batch(args.batch, ctx, vocab, gen, dev)
        opt.zero_grad()
        loss = net(x, y)
        loss.backward()
        opt.step()
        if step == 0:
            first = loss.item()
        if rank == 0 and (step + 1) % 10 == 0:
            print(f"step {step + 1}: loss {loss.item():.4f}", flush=True)
    final = loss.detach().clone()
    if ranks > 1:
        dist.all_reduce(final)
    if rank == 0:
        print(f"mean loss over {ranks} ranks: first {first:.4f}, last {final.item() / ranks:.4f}", flush=True)
    if args.generate and rank == 0:
        with torch.no_grad():
            seq = batch(1, ctx, vocab, gen, dev)[0][:, :8]
            for _ in range(args.generate):
                seq = torch.cat((seq, model(seq[:, -ctx:])[:, -1].argmax(-1, keepdim=True)), 1)
        print("generated", seq[0].tolist(), flush=True)
    env.barrier()
    env.close()


if __name__ == "__main__":
    main()
