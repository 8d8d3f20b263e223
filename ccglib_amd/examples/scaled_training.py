"""A small network trained and then asked with the 8-bit operators, next to the same network in torch:

    y = W2 relu(W1 x), fitted to a teacher of the same form.

    python -m ccglib_amd.examples.scaled_training [--width 1000 --hidden 2000 --out 500 --batch 4096 --steps 100]

Training: each product of the layers, forward and backward, is a ScaledLinear; the update of a weight matrix is its
momentum, made nearly orthogonal by Orthogonalize. Answering: the trained weights are converted once by Quantize, with a
scale for each 128 x 128 values, and a single x at a time is multiplied with them by ScaledGEMM. What is printed: the loss
of both networks along the way, and how far the single answers are from those that the trained weights give in 64 bits.
"""
import argparse
import math
import time

import torch

import ccglib_amd as cc

VT = cc.ValueType


def stream():
    return torch.cuda.current_stream().cuda_stream


class ScaledProducts:
    """One layer's products in 8 bits."""

    def __init__(self, batch, w):
        out, width = w.shape
        self.linear = cc.ScaledLinear(batch, out, width, w.device.index, stream())
        self.y = torch.empty((batch, out), dtype=torch.bfloat16, device=w.device)
        self.dx = torch.empty((batch, width), dtype=torch.bfloat16, device=w.device)
        self.dw = torch.empty_like(w)
        self.weights = torch.empty_like(w, dtype=torch.bfloat16)

    def forward(self, w, x):
        self.weights.copy_(w)
        self.linear.SetWeights(self.weights.data_ptr())
        self.linear.Forward(x.data_ptr(), self.y.data_ptr())
        return self.y

    def backward(self, dy, first):
        self.linear.Backward(dy.data_ptr(), 0 if first else self.dx.data_ptr(), self.dw.data_ptr())
        return self.dx, self.dw


class TorchProducts:
    """The same in bfloat16, by torch."""

    def __init__(self, batch, w):
        pass

    def forward(self, w, x):
        self.w, self.x = w.bfloat16(), x
        return x @ self.w.t()

    def backward(self, dy, first):
        return dy @ self.w, (dy.t() @ self.x).float()


class OrthogonalUpdate:
    """W -= rate max(1, rows / columns)^(1/2) orthogonalised(momentum)."""

    def __init__(self, w):
        rows, columns = w.shape
        self.momentum = torch.zeros_like(w)
        self.update = torch.empty_like(w)
        self.scale = math.sqrt(max(1.0, rows / columns))
        self.orthogonalize = cc.Orthogonalize(1, rows, columns, w.device.index, stream(), VT.float32)

    def step(self, w, dw, rate):
        self.momentum.mul_(0.9).add_(dw)
        self.orthogonalize.Run(self.momentum.data_ptr(), self.update.data_ptr())
        w.sub_(self.update, alpha=rate * self.scale)


def train(products, width, hidden, out, batch, steps, seed=0, rate=0.02, report=None):
    """Losses of all steps, and the trained weights (float32)."""
    device = torch.device("cuda", torch.cuda.current_device())
    rng = torch.Generator(device=device).manual_seed(seed)

    def normal(rows, columns, scale=1.0):
        return torch.randn((rows, columns), device=device, generator=rng) * scale

    teacher = [normal(hidden, width, (2.0 / width) ** 0.5), normal(out, hidden, hidden ** -0.5)]
    weights = [normal(hidden, width, (2.0 / width) ** 0.5), normal(out, hidden, hidden ** -0.5)]
    layers = [products(batch, w) for w in weights]
    updates = [OrthogonalUpdate(w) for w in weights]
    losses = []
    for step in range(steps):
        x = normal(batch, width).bfloat16()
        target = torch.relu(x.float() @ teacher[0].t()) @ teacher[1].t()
        h = torch.relu(layers[0].forward(weights[0], x))
        error = layers[1].forward(weights[1], h).float() - target
        losses.append((error * error).mean())
        dy = (error * (2.0 / batch)).bfloat16()
        dh, dw1 = layers[1].backward(dy, first=False)
        _, dw0 = layers[0].backward(torch.where(h > 0, dh, torch.zeros_like(dh)), first=True)
        for w, dw, update in zip(weights, (dw0, dw1), updates):
            update.step(w, dw, rate * (1.0 - step / steps))
        if report and (step % report == 0 or step == steps - 1):
            print("  step %4d  loss %.5f" % (step, float(losses[-1])), flush=True)
    return [float(loss) for loss in losses], weights


class Answer:
    """y = W2 relu(W1 x) of one x at a time, the weights in 8 bits with a scale for each 128 x 128."""

    def __init__(self, weights):
        device = weights[0].device
        index = device.index
        self.layers = []
        for w in weights:
            out, width = w.shape
            pitch, down = cc.scaled_pitch(width), -(-width // 128)
            values = torch.empty((out, pitch), dtype=torch.uint8, device=device)
            scales = torch.empty((down, cc.scaled_pitch(-(-out // 128))), device=device)
            convert = cc.Quantize(1, out, width, index, stream(), VT.bfloat16, group=cc.ScaleGroup.blocks)
            kept = w.bfloat16()
            convert.Run(kept.data_ptr(), values.data_ptr(), scales.data_ptr())
            self.layers.append({
                "w": values, "scales": scales,
                "x": torch.empty((1, pitch), dtype=torch.uint8, device=device),
                "x_scales": torch.empty((down, cc.scaled_pitch(1)), device=device),
                "y": torch.empty((1, out), dtype=torch.bfloat16, device=device),
                "convert": cc.Quantize(1, 1, width, index, stream(), VT.bfloat16),
                "product": cc.ScaledGEMM(1, 1, out, width, index, stream())})

    def __call__(self, x):
        for i, layer in enumerate(self.layers):
            if i:
                x = torch.relu(x)
            layer["convert"].Run(x.data_ptr(), layer["x"].data_ptr(), layer["x_scales"].data_ptr())
            layer["product"].Run(layer["x"].data_ptr(), layer["x_scales"].data_ptr(), layer["w"].data_ptr(),
                                 layer["scales"].data_ptr(), layer["y"].data_ptr())
            x = layer["y"]
        return x


def answer_error(weights, count=8, seed=1):
    """|answers - those of the weights in 64 bits| / |those|, over `count` single inputs."""
    device = weights[0].device
    rng = torch.Generator(device=device).manual_seed(seed)
    answer, off, norm = Answer(weights), 0.0, 0.0
    for _ in range(count):
        x = torch.randn((1, weights[0].shape[1]), device=device, generator=rng).bfloat16()
        want = torch.relu(x.double() @ weights[0].double().t()) @ weights[1].double().t()
        got = answer(x).double()
        off += float((got - want).square().sum())
        norm += float(want.square().sum())
    return math.sqrt(off / norm)


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--width", type=int, default=1000)
    parser.add_argument("--hidden", type=int, default=2000)
    parser.add_argument("--out", type=int, default=500)
    parser.add_argument("--batch", type=int, default=4096)
    parser.add_argument("--steps", type=int, default=100)
    parser.add_argument("--report", type=int, default=20)
    args = parser.parse_args()
    sizes = (args.width, args.hidden, args.out, args.batch, args.steps)
    for name, products in (("8-bit products", ScaledProducts), ("bfloat16, torch", TorchProducts)):
        print(name)
        train(products, *sizes[:-1], 3)          # (what loads kernels)
        torch.cuda.synchronize()
        began = time.perf_counter()
        losses, weights = train(products, *sizes, report=args.report)
        torch.cuda.synchronize()
        print("  %.2f ms a step, with what both share" % (1e3 * (time.perf_counter() - began) / args.steps))
        if products is ScaledProducts:
            trained = weights
    print("single answers in 8 bits: %.4f of their size off" % answer_error(trained))


if __name__ == "__main__":
    main()
