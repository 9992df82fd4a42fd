#!/usr/bin/env python
"""A windowed model learns from a full-attention one: rotary positions, attention to a window and the first tokens, shared key/value
heads, the loss from the teacher's top logits; then it writes a few tokens from caches of fixed size.  Synthetic token ids, random
teacher, one GPU.

    python bench/distill_window.py --layers 4 --d_model 1024 --nheads 8 --kv-heads 2 --seqlen 3000 --window 512 --steps 10
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def main(argv=None):
    p = argparse.ArgumentParser()
    p.add_argument("--layers", type=int, default=2)
    p.add_argument("--d_model", type=int, default=512)
    p.add_argument("--nheads", type=int, default=4)
    p.add_argument("--kv-heads", type=int, default=2)
    p.add_argument("--ffn", type=int, default=0)
    p.add_argument("--vocab", type=int, default=1000)
    p.add_argument("--seqlen", type=int, default=640)
    p.add_argument("--window", type=int, default=128)
    p.add_argument("--sinks", type=int, default=4)
    p.add_argument("--theta", type=float, default=10000.0)
    p.add_argument("--scale-factor", type=float, default=1.0, help="context beyond the trained length, by parts")
    p.add_argument("--top", type=int, default=32)
    p.add_argument("--temperature", type=float, default=2.0)
    p.add_argument("--hard-weight", type=float, default=0.1)
    p.add_argument("--batchsize", type=int, default=4)
    p.add_argument("--micro-batch", type=int, default=2)
    p.add_argument("--steps", type=int, default=10)
    p.add_argument("--lr", type=float, default=1e-3)
    p.add_argument("--write", type=int, default=16, help="tokens to write at the end")
    a = p.parse_args(argv)
    torch.cuda.set_device(0)
    from meshslice_b200.models.decode import GPTDecoder
    from meshslice_b200.models.gpt import GPTConfig, GPTModel
    from meshslice_b200.ops.rotary import RotaryConfig
    from meshslice_b200.parallel.engine import LocalGemmEngine
    from meshslice_b200.parallel.mesh import EmuMesh
    from meshslice_b200.trainer import TrainConfig, Trainer

    device = torch.device("cuda", 0)
    rotary = RotaryConfig(head_dim=a.d_model // a.nheads, theta=a.theta, scaling="by_parts" if a.scale_factor > 1 else "none",
                          factor=a.scale_factor, original_len=a.seqlen)
    base = dict(n_layers=a.layers, d_model=a.d_model, n_heads=a.nheads, ffn=a.ffn or 4 * a.d_model, vocab=a.vocab, seq=a.seqlen,
                vocab_pad=256, rotary=rotary)
    mesh = EmuMesh(1, 1)
    LocalGemmEngine(mesh)
    teacher = GPTModel(mesh, GPTConfig(**base, init_std=0.05), device=device)
    student = Trainer(GPTConfig(**base, kv_heads=a.kv_heads, window=a.window, sinks=a.sinks),
                      TrainConfig(global_batch=a.batchsize, micro_batch=a.micro_batch, lr=a.lr), mesh_shape=(1, 1), device=device)
    ids = torch.randint(0, a.vocab, (a.batchsize, a.seqlen + 1), generator=torch.Generator().manual_seed(1)).pin_memory()
    losses = []
    for step in range(a.steps):
        losses.append(student.train_step(ids, teacher=lambda tok: teacher.top_logits(tok, a.top, a.temperature, a.hard_weight)))
        print(f"step {step + 1}: distillation loss {losses[-1]:.4f}")
    student.check()
    tokens = ids[:, :min(a.seqlen, 100)].to(device)
    decoder = GPTDecoder(student.model, a.batchsize)
    last, pos = decoder.prefill(tokens).argmax(1), tokens.shape[1]
    written = [last]
    for i in range(a.write - 1):
        last = decoder.step(last, torch.full((a.batchsize,), pos + i, dtype=torch.int64, device=device)).argmax(1)
        written.append(last)
    student.check()
    written = torch.stack(written, 1).tolist()
    print("written:", written[0])
    return losses, written


if __name__ == "__main__":
    main()
