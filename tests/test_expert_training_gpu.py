"""The example of a network with a layer of experts: it runs, and its gradients are those that autograd gives in 64 bits."""
import pytest
import torch

from ccglib_amd.examples.expert_training import ExpertNetwork, train

pytestmark = pytest.mark.gpu


def test_it_runs():
    losses, network = train(width=64, hidden=96, experts=5, chosen=2, batch=130, steps=3)
    assert len(losses) == 3 and all(v == v and v < float("inf") for v in losses)
    assert int(network.offsets[-1]) == 260


def test_gradients():
    """The longest way from dy back to w1 has eleven roundings to bfloat16 of what stands between (on the way there a, h, xs, b,
    ys, y; back dys, db, dz2, dxs, dh, da, dz1; z1 and z2 where act' is taken): 16 of them at most, each of a norm of 2^-9 of what is
    rounded (an error uniform in half a step of 2^-8, relative to values spread over a factor of two), independent of each other. The
    router's way (logits to dlogits) adds two more. Together below sqrt(18) 2^-9, and each may be enlarged by the layers behind it, which
    have gains of about 1 (weights of 1 / sqrt(width)): a factor of 4 is left for that."""
    batch, width, hidden, experts, chosen = 96, 64, 128, 4, 2
    network = ExpertNetwork(batch, width, hidden, experts, chosen)
    generator = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((batch, width), device="cuda", generator=generator).bfloat16()
    dy = torch.randn((batch, width), device="cuda", generator=generator).bfloat16()
    y = network.forward(x).clone()
    dx = network.backward(x, dy).clone()
    torch.cuda.synchronize()
    w = {name: v.double().cpu().requires_grad_(True) for name, v in network.held.items()}
    x64 = x.double().cpu().requires_grad_(True)
    h = x64 + torch.nn.functional.gelu(x64 @ w["w1"].t() + w["b1"], approximate="tanh") @ w["w2"].t() + w["b2"]
    logits = h @ w["router"].t()
    # (the network's own choice: logits that are nearly the same may be ordered by their rounding)
    numbers = network.numbers.long().cpu()
    share = torch.softmax(logits.gather(1, numbers), dim=1)
    out = torch.zeros((batch, width), dtype=torch.float64)
    for j in range(chosen):
        z = torch.bmm(w["v1"][numbers[:, j]], h[:, :, None])
        out = out + share[:, j:j + 1] * torch.bmm(w["v2"][numbers[:, j]], z * torch.sigmoid(z))[:, :, 0]
    (out * dy.double().cpu()).sum().backward()
    bound = 4 * 18 ** 0.5 * 2.0 ** -9
    pairs = {"y": (y, out.detach()), "dx": (dx, x64.grad)} | {n: (network.gradients[n], v.grad) for n, v in w.items()}
    for name, (got, want) in pairs.items():
        off = float((got.double().cpu() - want).norm() / want.norm())
        assert off <= bound, "%s: %.4f" % (name, off)
