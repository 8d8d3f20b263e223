"""A small network with a layer of experts, trained with the 16-bit layers:

    h = x + W2 gelu(W1 x + b1) + b2
    y = sum over the k experts that a router chooses of  weight  V2[e] silu(V1[e] h)

fitted to a teacher of the same form.

    python -m ccglib_amd.examples.expert_training [--width 512 --hidden 1024 --experts 16 --chosen 2 --batch 4096 --steps 200]

Each product with what stands around it is one call of FusedLinear, those of all experts one of GroupedLinear; Route
chooses, and Combine brings rows to their experts and back. Weights are kept in 32 bits, layers have them in bfloat16. What is
printed: the loss along the way, how the rows spread over the experts, and the time of a step.
"""
import argparse
import time

import torch

import ccglib_amd as cc

VT, ACT = cc.ValueType, cc.Activation


class ExpertNetwork:
    """The layers and their buffers for batches of one size. Gradients are those of the last backward()."""

    def __init__(self, batch, width, hidden, experts, chosen, seed=0, device=None):
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        index, stream = self.device.index, torch.cuda.current_stream(self.device).cuda_stream
        rows = batch * chosen
        generator = torch.Generator(device=self.device).manual_seed(seed)

        def normal(*shape):
            return torch.randn(shape, device=self.device, generator=generator) * shape[-1] ** -0.5

        self.weights = {"w1": normal(hidden, width), "w2": normal(width, hidden), "router": normal(experts, width),
                        "v1": normal(experts, hidden, width), "v2": normal(experts, width, hidden),
                        "b1": torch.zeros(hidden, device=self.device), "b2": torch.zeros(width, device=self.device)}
        self.gradients = {name: torch.empty_like(w) for name, w in self.weights.items()}
        self.held = {name: w.bfloat16() for name, w in self.weights.items()}
        self.layers = {
            "1": cc.FusedLinear(batch, hidden, width, index, stream, VT.bfloat16, ACT.gelu),
            "2": cc.FusedLinear(batch, width, hidden, index, stream),
            "router": cc.FusedLinear(batch, experts, width, index, stream),
            "v1": cc.GroupedLinear(experts, rows, hidden, width, index, stream, VT.bfloat16, ACT.silu),
            "v2": cc.GroupedLinear(experts, rows, width, hidden, index, stream)}
        self.route = cc.Route(batch, experts, chosen, index, stream, VT.bfloat16)
        self.combine = cc.Combine(batch, chosen, width, index, stream)

        def half(*shape):
            return torch.empty(shape, dtype=torch.bfloat16, device=self.device)

        def whole(*shape):
            return torch.empty(shape, dtype=torch.int32, device=self.device)

        self.a, self.z1, self.da = half(batch, hidden), half(batch, hidden), half(batch, hidden)
        self.h, self.y, self.dh = (half(batch, width) for _ in range(3))
        self.logits, self.dlogits = half(batch, experts), half(batch, experts)
        self.numbers, self.slots, self.offsets = whole(batch, chosen), whole(batch, chosen), whole(experts + 1)
        self.share, self.dshare = (torch.empty((batch, chosen), device=self.device) for _ in range(2))
        self.xs, self.dxs, self.ys, self.dys = (half(rows, width) for _ in range(4))
        self.b, self.z2, self.db = (half(rows, hidden) for _ in range(3))
        self.dh_router, self.dx = half(batch, width), half(batch, width)

    def forward(self, x):
        p, w, at = self.layers, self.held, (lambda t: t.data_ptr())
        p["1"].Forward(at(x), at(w["w1"]), at(w["b1"]), 0, at(self.a), at(self.z1))
        p["2"].Forward(at(self.a), at(w["w2"]), at(w["b2"]), at(x), at(self.h))
        p["router"].Forward(at(self.h), at(w["router"]), 0, 0, at(self.logits))
        self.route.Run(at(self.logits), at(self.numbers), at(self.share), at(self.offsets), at(self.slots))
        self.combine.Spread(at(self.h), at(self.slots), 0, at(self.xs))
        p["v1"].Forward(at(self.xs), at(self.offsets), at(w["v1"]), 0, 0, at(self.b), at(self.z2))
        p["v2"].Forward(at(self.b), at(self.offsets), at(w["v2"]), 0, 0, at(self.ys))
        self.combine.Run(at(self.ys), at(self.slots), at(self.share), at(self.y))
        return self.y

    def backward(self, x, dy):
        p, w, g, at = self.layers, self.held, self.gradients, (lambda t: t.data_ptr())
        self.combine.Backward(at(dy), at(self.ys), at(self.slots), at(self.share), at(self.dys), at(self.dshare))
        p["v2"].Backward(at(self.dys), 0, at(self.b), at(self.offsets), at(w["v2"]), at(self.db), at(g["v2"]))
        p["v1"].Backward(at(self.db), at(self.z2), at(self.xs), at(self.offsets), at(w["v1"]), at(self.dxs), at(g["v1"]))
        self.combine.Run(at(self.dxs), at(self.slots), 0, at(self.dh))
        self.route.Backward(at(self.logits), at(self.numbers), at(self.share), at(self.dshare), at(self.dlogits))
        p["router"].Backward(at(self.dlogits), 0, at(self.h), at(w["router"]), at(self.dh_router), at(g["router"]))
        self.dh.add_(self.dh_router)
        p["2"].Backward(at(self.dh), 0, at(self.a), at(w["w2"]), at(self.da), at(g["w2"]), at(g["b2"]))
        p["1"].Backward(at(self.da), at(self.z1), at(x), at(w["w1"]), at(self.dx), at(g["w1"]), at(g["b1"]))
        return self.dx.add_(self.dh)          # (x goes into h as it is, too)

    def step(self, rate):
        for name, w in self.weights.items():
            w.sub_(self.gradients[name], alpha=rate)
            self.held[name].copy_(w)


def train(width, hidden, experts, chosen, batch, steps, rate=1.0, seed=0, report=None):
    """Losses of all steps, and the trained network."""
    network = ExpertNetwork(batch, width, hidden, experts, chosen, seed)
    teacher = ExpertNetwork(batch, width, hidden, experts, chosen, seed + 1)
    generator = torch.Generator(device=network.device).manual_seed(seed + 2)
    losses = []
    for step in range(steps):
        x = torch.randn((batch, width), device=network.device, generator=generator).bfloat16()
        error = network.forward(x).float() - teacher.forward(x).float()
        losses.append((error * error).mean())
        network.backward(x, (error * (2.0 / error.numel())).bfloat16())
        network.step(rate)
        if report and (step % report == 0 or step == steps - 1):
            print("  step %4d  loss %.5f" % (step, float(losses[-1])), flush=True)
    return [float(loss) for loss in losses], network


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--width", type=int, default=512)
    parser.add_argument("--hidden", type=int, default=1024)
    parser.add_argument("--experts", type=int, default=16)
    parser.add_argument("--chosen", type=int, default=2)
    parser.add_argument("--batch", type=int, default=4096)
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--rate", type=float, default=1.0)
    parser.add_argument("--report", type=int, default=40)
    args = parser.parse_args()
    sizes = (args.width, args.hidden, args.experts, args.chosen, args.batch)
    train(*sizes, 3)          # (what loads kernels)
    torch.cuda.synchronize()
    began = time.perf_counter()
    _, network = train(*sizes, args.steps, args.rate, report=args.report)
    torch.cuda.synchronize()
    print("  %.2f ms a step, the teacher's forward pass among it" % (1e3 * (time.perf_counter() - began) / args.steps))
    counts = network.offsets.diff()
    print("rows of an expert: %d to %d" % (int(counts.min()), int(counts.max())))


if __name__ == "__main__":
    main()
