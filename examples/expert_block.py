"""A small stack of sparse feed-forward blocks made of this library's RMS norm, expert router, token sort and experts'
products: trained, then run once more with rows and matrices in 8 bits.

    python examples/expert_block.py

Each block is   h = h + sum over the chosen experts e of weight_e * down_e(silu(gate_e n) * up_e n),   n = RMS norm(h).
The router's choices put the tokens in the order of their experts, so that the products of all experts are one call, and
the weighted sum and the residual are another.  No call waits for the number of rows that an expert has.  Gradients of
gradients are not computed: asking for them is an error."""
from __future__ import annotations

import os
import sys

import torch
from torch.autograd.function import once_differentiable

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import lc_parallel_primitive_amd as lcpp  # noqa: E402

EPS = 1e-6
NORM, ROUTER, ORDER, PRODUCT = lcpp.DeviceRMSNorm(), lcpp.DeviceExpertRouter(), lcpp.DeviceTokenSort(), lcpp.DeviceExpertProduct()


def _temp(nbytes):
    return torch.empty(nbytes, dtype=torch.uint8, device="cuda") if nbytes else None


class Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w):
        y, rstd = torch.empty_like(x), torch.empty(x.shape[0], device=x.device)
        NORM.Forward(x, y, w, EPS, rstd)
        ctx.save_for_backward(x, w, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, rstd = ctx.saved_tensors
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        temp = _temp(lcpp.DeviceRMSNorm.GetBackwardTempStorageBytes(x.dtype, *x.shape))
        NORM.Backward(temp, dy.contiguous(), x, w, rstd, dx, dw)
        return dx, dw


class Route(torch.autograd.Function):
    """(the experts of each row of logits, their weights)"""

    @staticmethod
    def forward(ctx, logits, choices):
        experts = torch.empty(logits.shape[0], choices, dtype=torch.int32, device=logits.device)
        weights = torch.empty(logits.shape[0], choices, device=logits.device)
        ROUTER.Forward(logits, experts, weights)
        ctx.save_for_backward(logits, experts)
        ctx.mark_non_differentiable(experts)
        return experts, weights

    @staticmethod
    @once_differentiable
    def backward(ctx, _, dw):
        logits, experts = ctx.saved_tensors
        dl = torch.empty_like(logits)
        ROUTER.Backward(logits, experts, dw.contiguous(), dl)
        return dl, None


class Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions):
        rows = torch.empty(positions.numel(), x.shape[1], dtype=x.dtype, device=x.device)
        ORDER.Dispatch(x, positions, rows)
        ctx.save_for_backward(positions)
        return rows

    @staticmethod
    @once_differentiable
    def backward(ctx, dr):
        (positions,) = ctx.saved_tensors
        dx = torch.empty(positions.shape[0], dr.shape[1], dtype=dr.dtype, device=dr.device)
        ORDER.DispatchBackward(dr.contiguous(), positions, dx)
        return dx, None


class Product(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, matrices, offsets):
        y = torch.empty(rows.shape[0], matrices.shape[1], dtype=rows.dtype, device=rows.device)
        PRODUCT.Forward(rows, matrices, offsets, y)
        ctx.save_for_backward(rows, matrices, offsets)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        rows, matrices, offsets = ctx.saved_tensors
        dx, dm = torch.empty_like(rows), torch.empty_like(matrices)
        PRODUCT.Backward(dy.contiguous(), rows, matrices, offsets, dx, dm)
        return dx, dm, None


class Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, residual, positions):
        out = torch.empty_like(residual)
        ORDER.Combine(rows, positions, weights, out, residual)
        ctx.save_for_backward(rows, weights, positions)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        rows, weights, positions = ctx.saved_tensors
        dr, dw = torch.empty_like(rows), torch.empty_like(weights)
        dy = dy.contiguous()
        ORDER.CombineBackward(dy, rows, positions, weights, dr, dw)
        return dr, dw, dy, None


def eight_bits(m):
    """(values, scales) of matrices (experts, outputs, inputs): one scale for each 128 x 128 of them."""
    e, o, i = m.shape
    po, pi = -(-o // 128), -(-i // 128)
    wide = torch.zeros(e, po * 128, pi * 128, device=m.device)
    wide[:, :o, :i] = m
    blocks = wide.view(e, po, 128, pi, 128)
    scales = blocks.abs().amax((2, 4)).clamp(min=2.0**-100) / 448
    values = (blocks / scales[:, :, None, :, None]).view_as(wide)[:, :o, :i]
    return values.to(torch.float8_e4m3fn).contiguous(), scales


class Model(torch.nn.Module):
    def __init__(self, vocab=64, width=256, hidden=160, experts=8, choices=2, layers=2, dtype=torch.bfloat16, seed=1):
        super().__init__()
        torch.manual_seed(seed)
        self.layers, self.experts, self.choices, self.dtype = layers, experts, choices, dtype

        def matrix(*shape):
            return torch.nn.Parameter(torch.randn(*shape, device="cuda") * shape[-1] ** -0.5)

        self.embed = torch.nn.Parameter(torch.randn(vocab, width, device="cuda"))
        self.router = torch.nn.ParameterList(matrix(experts, width) for _ in range(layers))
        # gate and up are the halves of one product
        self.up = torch.nn.ParameterList(matrix(experts, 2 * hidden, width) for _ in range(layers))
        self.down = torch.nn.ParameterList(matrix(experts, width, hidden) for _ in range(layers))
        self.norm = torch.nn.ParameterList(torch.nn.Parameter(torch.ones(width, device="cuda")) for _ in range(layers + 1))
        self.head = matrix(vocab, width)
        self.chosen = []  # of the last forward pass, for each layer

    def _sort(self, experts):
        positions = torch.empty_like(experts)
        offsets = torch.empty(self.experts + 1, dtype=torch.int32, device="cuda")
        temp = _temp(lcpp.DeviceTokenSort.GetTempStorageBytes(*experts.shape, self.experts))
        ORDER.Sort(temp, experts, self.experts, positions, offsets)
        return positions, offsets

    def forward(self, tokens):
        h = self.embed[tokens].to(self.dtype)
        self.chosen = []
        for i in range(self.layers):
            normed = Norm.apply(h, self.norm[i])
            experts, weights = Route.apply(normed.float() @ self.router[i].t(), self.choices)
            positions, offsets = self._sort(experts)
            self.chosen.append(experts)
            gate, up = Product.apply(Dispatch.apply(normed, positions), self.up[i].to(self.dtype), offsets).chunk(2, 1)
            rows = Product.apply(torch.nn.functional.silu(gate) * up, self.down[i].to(self.dtype), offsets)
            h = Combine.apply(rows, weights, h, positions)
        return Norm.apply(h, self.norm[self.layers]).float() @ self.head.t()

    @torch.no_grad()
    def in_eight_bits(self):
        """The matrices of every block in 8 bits, laid out once."""
        return [(eight_bits(self.up[i]), eight_bits(self.down[i])) for i in range(self.layers)]

    @torch.no_grad()
    def serve(self, tokens, matrices):
        """The logits with the experts' rows and matrices in 8 bits: the norm writes its rows' values and scales itself."""
        h = self.embed[tokens].to(self.dtype)
        n, width = h.shape
        pairs = n * self.choices
        self.chosen = []
        rows = None
        for i in range(self.layers):
            (up, up_scales), (down, down_scales) = matrices[i]
            groups = up_scales.shape[2]
            normed, total = torch.empty_like(h), torch.empty_like(h)
            values, scales = torch.empty(n, width, dtype=up.dtype, device="cuda"), torch.empty(n, groups, device="cuda")
            if rows is None:
                NORM.Forward(h, normed, self.norm[i], EPS, None, values, scales)
            else:  # the sum of the block before, and its norm
                NORM.AddForward(rows, h, total, normed, self.norm[i], EPS, None, values, scales)
                h = total
            experts = torch.empty(n, self.choices, dtype=torch.int32, device="cuda")
            weights = torch.empty(n, self.choices, device="cuda")
            ROUTER.Forward(normed.float() @ self.router[i].t(), experts, weights)
            self.chosen.append(experts)
            positions, offsets = self._sort(experts)
            sorted_values = torch.empty(pairs, width, dtype=up.dtype, device="cuda")
            sorted_scales = torch.empty(pairs, groups, device="cuda")
            ORDER.Dispatch(values, positions, sorted_values)
            ORDER.Dispatch(scales, positions, sorted_scales)
            both = torch.empty(pairs, up.shape[1], dtype=self.dtype, device="cuda")
            PRODUCT.Forward(sorted_values, up, offsets, both, sorted_scales, up_scales)
            gate, upper = both.chunk(2, 1)
            inner, inner_scales = _rows_in_eight_bits(torch.nn.functional.silu(gate) * upper)
            results = torch.empty(pairs, width, dtype=self.dtype, device="cuda")
            PRODUCT.Forward(inner, down, offsets, results, inner_scales, down_scales)
            rows = torch.empty_like(h)
            ORDER.Combine(results, positions, weights, rows)
        normed, total = torch.empty_like(h), torch.empty_like(h)
        if rows is None:
            NORM.Forward(h, normed, self.norm[0], EPS)
        else:
            NORM.AddForward(rows, h, total, normed, self.norm[self.layers], EPS)
        return normed.float() @ self.head.t()


def _rows_in_eight_bits(x):
    n, cols = x.shape
    parts = -(-cols // 128)
    wide = torch.zeros(n, parts * 128, device=x.device)
    wide[:, :cols] = x
    groups = wide.view(n, parts, 128)
    scales = groups.abs().amax(2).clamp(min=2.0**-100) / 448
    return (groups / scales[:, :, None]).view(n, -1)[:, :cols].to(torch.float8_e4m3fn).contiguous(), scales


def train(model, steps=60, tokens=512, lr=3e-3, seed=0):
    """The loss of every step: the next of a token is another one, always the same."""
    g = torch.Generator()
    g.manual_seed(seed)
    vocab = model.embed.shape[0]
    after = torch.randperm(vocab, generator=g).cuda()
    optimizer = torch.optim.Adam(model.parameters(), lr=lr)
    losses = []
    for _ in range(steps):
        x = torch.randint(0, vocab, (tokens,), generator=g).cuda()
        loss = torch.nn.functional.cross_entropy(model(x), after[x])
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
    return losses


if __name__ == "__main__":
    net = Model()
    history = train(net)
    print(f"loss {history[0]:.3f} -> {history[-1]:.3f} in {len(history)} steps")
    every = torch.arange(net.embed.shape[0], device="cuda")
    with torch.no_grad():
        want = net(every)
    got = net.serve(every, net.in_eight_bits())
    print(f"rows and matrices in 8 bits: logits within {float((got - want).norm() / want.norm()):.2e} of the others'")
