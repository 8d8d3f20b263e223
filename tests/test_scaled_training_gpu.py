"""The example that trains with ScaledLinear and Orthogonalize and answers with Quantize and ScaledGEMM."""
import pytest

torch = pytest.importorskip("torch")

from ccglib_amd.examples import scaled_training as example

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width,hidden,out,batch", [(130, 260, 65, 300), (256, 512, 128, 1024)])
def test_it_learns_as_the_same_network_in_torch_does(width, hidden, out, batch):
    losses, weights = example.train(example.ScaledProducts, width, hidden, out, batch, 60)
    plain, _ = example.train(example.TorchProducts, width, hidden, out, batch, 60)
    assert losses[-1] < 0.5 * losses[0]
    # (a value of 8 bits is at most 2^-4 off, so a product of independent ones about 5 %, and its square adds less than
    # a hundredth of the outputs' mean square, which is about 1, to a loss)
    assert losses[-1] < 1.1 * plain[-1] + 0.02
    # (2^-4 / sqrt(3) for a value, two values a product, two layers: 0.072)
    assert example.answer_error(weights) < 0.08
