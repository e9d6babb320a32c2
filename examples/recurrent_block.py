"""A small recurrent language model made of this library's layer norm, gated recurrence and dropout: trained on
sequences that count in steps of their own, then decoded one token at a time.

    python examples/recurrent_block.py

Each residual block is   h = h + dropout(W_o recurrence(W_g n, W_v n)),   n = layer norm(h),   and a block's
residual sum, dropout and the next block's norm are one call.  Training packs sequences of different lengths one
behind the other (begin and end offsets, nothing padded); decoding keeps one state per layer and sequence in a pool
of slots and gives the same logits as the whole sequences at once.  Gradients of gradients are not computed: asking
for them is an error."""
from __future__ import annotations

import os
import sys

import torch
from torch.autograd.function import once_differentiable

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import lc_parallel_primitive_amd as lcpp  # noqa: E402

EPS = 1e-5
NORM, MIX = lcpp.DeviceLayerNorm(), lcpp.DeviceGatedRecurrence()


def _temp(nbytes):
    return torch.empty(nbytes, dtype=torch.uint8, device="cuda") if nbytes else None


class Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b):
        y = torch.empty_like(x)
        mean, rstd = (torch.empty(x.shape[0], device=x.device) for _ in range(2))
        NORM.Forward(x, y, w, b, EPS, mean, rstd)
        ctx.save_for_backward(x, w, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, mean, rstd = ctx.saved_tensors
        dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
        temp = _temp(lcpp.DeviceLayerNorm.GetBackwardTempStorageBytes(x.dtype, *x.shape))
        NORM.Backward(temp, dy.contiguous(), x, w, mean, rstd, dx, dw, db)
        return dx, dw, db


class AddNorm(torch.autograd.Function):
    """(residual + dropout(x), its layer norm)"""

    @staticmethod
    def forward(ctx, x, residual, w, b, p, seed, offset):
        total, y = torch.empty_like(x), torch.empty_like(x)
        mean, rstd = (torch.empty(x.shape[0], device=x.device) for _ in range(2))
        NORM.AddForward(x, residual, total, y, w, b, EPS, mean, rstd, p=p, seed=seed, offset=offset)
        ctx.save_for_backward(total, w, mean, rstd)
        ctx.drop = dict(p=p, seed=seed, offset=offset)  # all that the backward pass needs of the mask
        return total, y

    @staticmethod
    @once_differentiable
    def backward(ctx, dtotal, dy):
        total, w, mean, rstd = ctx.saved_tensors
        dres, dx = torch.empty_like(total), torch.empty_like(total)
        dw, db = torch.empty_like(w), torch.empty_like(w)
        temp = _temp(lcpp.DeviceLayerNorm.GetBackwardTempStorageBytes(total.dtype, *total.shape))
        NORM.AddBackward(temp, dy.contiguous(), dtotal.contiguous(), total, w, mean, rstd, dres, dx, dw, db, **ctx.drop)
        return dx, dres, dw, db, None, None, None


class Recurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, x, begin, end, longest):
        n, (rows, c) = begin.numel(), x.shape
        y = torch.empty_like(x)
        ctx.temp = _temp(lcpp.DeviceGatedRecurrence.GetTempStorageBytes(n, longest, c, rows))
        saved = torch.empty(lcpp.DeviceGatedRecurrence.GetPackedCheckpointRows(n, longest, rows), c, device=x.device)
        ctx.where = dict(d_begin_offsets=begin, d_end_offsets=end, max_length=longest)
        MIX.Forward(ctx.temp, gate, x, y, "sigmoid", d_checkpoints=saved, **ctx.where)
        ctx.save_for_backward(gate, x, saved)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        gate, x, saved = ctx.saved_tensors
        dg, dx = torch.empty_like(dy), torch.empty_like(dy)
        MIX.Backward(ctx.temp, gate, x, saved, dy.contiguous(), dg, dx, "sigmoid", **ctx.where)
        return dg, dx, None, None, None


class Model(torch.nn.Module):
    def __init__(self, vocab=32, width=192, layers=2, p=0.1, seed=1):
        super().__init__()
        torch.manual_seed(seed)
        self.layers, self.width, self.p, self.seed, self.step = layers, width, p, seed, 0

        def matrix(rows, cols):
            return torch.nn.Parameter(torch.randn(rows, cols, device="cuda") * rows**-0.5)

        self.embed = torch.nn.Parameter(torch.randn(vocab, width, device="cuda"))
        # gate and value are the halves of one product
        self.mix_in = torch.nn.ParameterList(matrix(width, 2 * width) for _ in range(layers))
        self.mix_out = torch.nn.ParameterList(matrix(width, width) for _ in range(layers))
        self.norm_w = torch.nn.ParameterList(torch.nn.Parameter(torch.ones(width, device="cuda")) for _ in range(layers + 1))
        self.norm_b = torch.nn.ParameterList(torch.nn.Parameter(torch.zeros(width, device="cuda")) for _ in range(layers + 1))
        self.head = matrix(width, vocab)

    def forward(self, tokens, begin, end, longest):
        """The logits of packed sequences: tokens (rows,), begin and end offsets of each sequence."""
        p = self.p if self.training else 0.0
        self.step += self.training
        h = self.embed[tokens].bfloat16()
        normed = Norm.apply(h, self.norm_w[0], self.norm_b[0])
        for i in range(self.layers):
            gate, value = (normed @ self.mix_in[i].bfloat16()).split(self.width, 1)  # views: rows 2 * width apart
            mixed = Recurrence.apply(gate, value, begin, end, longest) @ self.mix_out[i].bfloat16()
            h, normed = AddNorm.apply(mixed, h, self.norm_w[i + 1], self.norm_b[i + 1], p, self.seed,
                                      self.step * self.layers + i)
        return normed.float() @ self.head

    @torch.no_grad()
    def decode(self, tokens, states, slots):
        """The logits after one more token of each sequence, whose states lie at `slots` of `states` (layers, pool,
        width) and are advanced in place."""
        h = self.embed[tokens].bfloat16()
        normed, total = torch.empty_like(h), torch.empty_like(h)
        NORM.Forward(h, normed, self.norm_w[0], self.norm_b[0], EPS)
        for i in range(self.layers):
            gate, value = (normed @ self.mix_in[i].bfloat16()).split(self.width, 1)
            mixed = torch.empty_like(h)
            MIX.Step(gate, value, states[i], states[i], mixed, "sigmoid", d_slots=slots)
            NORM.AddForward(mixed @ self.mix_out[i].bfloat16(), h, total, normed, self.norm_w[i + 1], self.norm_b[i + 1], EPS)
            h, total = total, torch.empty_like(h)
        return normed.float() @ self.head


def batch(generator, lengths, vocab):
    """Sequences that count in steps of their own, which the first two tokens tell.  (tokens, targets, begin, end,
    longest)"""
    start = torch.randint(0, vocab, (len(lengths),), generator=generator)
    stride = torch.randint(1, 4, (len(lengths),), generator=generator)
    rows = [(start[i] + stride[i] * torch.arange(n + 1)) % vocab for i, n in enumerate(lengths)]
    end = torch.tensor(lengths).cumsum(0).to(torch.int32)
    begin = end - torch.tensor(lengths, dtype=torch.int32)
    return (torch.cat([r[:-1] for r in rows]).cuda(), torch.cat([r[1:] for r in rows]).cuda(), begin.cuda(), end.cuda(),
            max(lengths))


def train(model, steps=60, lr=3e-3, seed=0):
    """The loss of every step."""
    g = torch.Generator()
    g.manual_seed(seed)
    optimizer = torch.optim.Adam(model.parameters(), lr=lr)
    losses = []
    model.train()
    for _ in range(steps):
        lengths = torch.randint(1, 200, (24,), generator=g).tolist()
        tokens, targets, begin, end, longest = batch(g, lengths, model.embed.shape[0])
        loss = torch.nn.functional.cross_entropy(model(tokens, begin, end, longest), targets)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
    return losses


@torch.no_grad()
def decoding_error(model, seed=5, lengths=(1, 9, 40, 33)):
    """How far the logits of single steps are from those of the whole sequences, relative to the largest."""
    g = torch.Generator()
    g.manual_seed(seed)
    model.eval()
    tokens, _, begin, end, longest = batch(g, list(lengths), model.embed.shape[0])
    whole = model(tokens, begin, end, longest)
    pool = 7
    states = torch.zeros(model.layers, pool, model.width, device="cuda")
    slots = torch.tensor([4, 0, 6, 2], dtype=torch.int32, device="cuda")
    worst = 0.0
    for t in range(longest):
        live = torch.tensor([t < n for n in lengths], device="cuda")
        at = (begin.long() + t).clamp(max=tokens.numel() - 1)
        # sequences that are done stay in the batch as padding
        logits = model.decode(tokens[at], states, torch.where(live, slots, -1).to(torch.int32))
        worst = max(worst, float((logits - whole[at])[live].abs().max()))
    return worst / float(whole.abs().max())


if __name__ == "__main__":
    net = Model()
    history = train(net)
    print(f"loss {history[0]:.3f} -> {history[-1]:.3f} in {len(history)} steps")
    print(f"decoding one token at a time: logits within {decoding_error(net):.2e} of the whole sequences'")
