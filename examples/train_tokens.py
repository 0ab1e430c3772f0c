"""A small next-token model trained through the layers and the 8-bit optimizer of this package.

    python examples/train_tokens.py [--steps 40]

Every step sums two micro-batches: table rows are looked up and scaled (`layers.embedding`), dropped, and go through blocks that
add a dropped branch to the residual and norm it in one kernel (`layers.rms_norm`); the loss is read off the bf16 logits as they are
(`losses.token_logprobs`, where a target outside the vocabulary counts for nothing).  The table's gradient is kept in float32
and accumulated over the micro-batches by `layers.embedding_grad`; the others come from autograd.  Both are what
`Adam8bit` reads as they are.  The text is synthetic: each token follows from the one before it.
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from eridiffusion_amd import layers, losses  # noqa: E402
from eridiffusion_amd.adam8bit import Adam8bit, Adam8bitConfig  # noqa: E402

VOCAB, DIM, BLOCKS, PAD = 1000, 256, 2, 0


def new(*shape, std):
    return (torch.randn(*shape, device="cuda") * std).bfloat16()


class Model:
    def __init__(self, p):
        self.p = p
        self.table = new(VOCAB, DIM, std=1 / math.sqrt(DIM))
        self.table.grad_dtype = None  # its gradient is float32
        self.up = [new(DIM, 4 * DIM, std=1 / math.sqrt(DIM)).requires_grad_() for _ in range(BLOCKS)]
        self.down = [new(4 * DIM, DIM, std=0.5 / math.sqrt(DIM)).requires_grad_() for _ in range(BLOCKS)]
        self.norms = [torch.ones(DIM, device="cuda", dtype=torch.bfloat16, requires_grad=True) for _ in range(BLOCKS + 1)]
        self.head = new(DIM, VOCAB, std=1 / math.sqrt(DIM)).requires_grad_()

    def parameters(self):
        return [self.table, self.head] + self.up + self.down + self.norms

    def loss(self, rows, target, step):
        """step numbers the micro-batch: each, and each place in the model, draws masks of its own."""
        h = layers.dropout(rows, self.p, seed=1, offset=step)
        y = layers.rms_norm(h, self.norms[0]).y
        for i in range(BLOCKS):
            branch = torch.nn.functional.gelu(y @ self.up[i]) @ self.down[i]
            y, h, _, _ = layers.rms_norm(branch, self.norms[i + 1], residual=h, p=self.p, seed=2 + i, offset=step)
        asked = (target >= 0) & (target < VOCAB)  # the others have log probability 0, and are not counted either
        return -losses.token_logprobs(y @ self.head, target).logprob.sum() / asked.sum()


def train(steps=40, batch=16, length=64, micro=2, p=0.1, seed=0, log=print):
    """Losses of the steps."""
    torch.manual_seed(seed)
    model, scale = Model(p), math.sqrt(DIM)
    opt = Adam8bit(model.parameters(), Adam8bitConfig(lr=2e-3, weight_decay=0.0))
    table_grad = torch.empty(VOCAB, DIM, device="cuda")
    follows = torch.randperm(VOCAB - 1, device="cuda") + 1  # of each token but the padding
    losses = []
    for step in range(steps):
        total = 0.0
        opt.zero_grad()
        for m in range(micro):
            ids = torch.randint(1, VOCAB, (batch, length), device="cuda")
            target = follows[ids - 1]
            ids[:, -8:] = PAD  # the ends of the sequences, which get no gradient and are not asked for
            rows = layers.embedding(ids, model.table, scale).requires_grad_()
            loss = model.loss(rows, torch.where(ids == PAD, -100, target), step * micro + m) / micro
            loss.backward()
            layers.embedding_grad(ids, rows.grad, VOCAB, scale, padding_id=PAD, out=table_grad, accumulate=m > 0)
            total += loss.detach()
        model.table.grad = table_grad
        opt.step()
        losses.append(float(total))
        if log and (step % 10 == 0 or step == steps - 1):
            log("step %3d  loss %.3f" % (step, losses[-1]))
    return losses


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=40)
    train(ap.parse_args().steps)
