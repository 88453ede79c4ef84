"""The encoder operators together, as the example uses them: train, index, search."""

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "encoder_search.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("encoder_search", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_trained_vectors_find_their_topic(example, dtype):
    """64 topics: by chance 1.6% of the neighbours are right. Half of them is far above what untrained vectors find."""
    before, after, first, last = example.run(texts=4096, steps=80, words=2048, dtype=dtype, report=lambda *_: None)
    assert before < 0.25 and after > 0.5
    assert first > 3.5 and last < 1.0


def test_one_step_follows_the_gradient_of_its_loss(example):
    """A step's weights against those that autograd's gradients give, in 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(1)
    tokens, topic = example.make_texts(200, 8, 300, 7, g)
    enc = example.Encoder(300, 24, 40, 16, 8, torch.float32, g)
    table, w, b = enc.table.double(), [x.double() for x in enc.weights], [x.double() for x in enc.biases]
    leaves = [table, *w, *b]
    for x in leaves:
        x.requires_grad_()
    found = torch.where(tokens[..., None] >= 0, table[tokens.clamp(min=0)], 0.0)
    h = torch.nn.functional.gelu((found.reshape(-1, 24) @ w[0].T + b[0]).view(200, 7, 40))
    loss = torch.nn.functional.cross_entropy((h.mean(1) @ w[1].T + b[1]) @ w[2].T + b[2], topic)
    grads = torch.autograd.grad(loss, leaves)

    got = enc.step(tokens, topic, 0.02, 10.0)
    # fp32 sums of at most 1,400 terms: 1e-5 of a result's largest entry leaves a factor of ten.
    assert abs(got.item() - loss.item()) < 1e-5 * loss.item()

    def near(x, y, scale):
        assert (x.double() - y).abs().max().item() <= 1e-5 * scale.abs().max().item()

    near(enc.table - table.detach().float(), -10.0 * grads[0], table.detach())
    for i in range(3):
        near(enc.momentum[i], 0.1 * grads[1 + i], 0.1 * grads[1 + i])
        near(enc.biases[i], -0.02 * grads[4 + i], 0.02 * grads[4 + i])
        # The step is the momentum orthogonalised: its singular values lie near one.
        step = (w[i].detach() - enc.weights[i].double()) / 0.02 / max(1.0, w[i].shape[0] / w[i].shape[1]) ** 0.5
        assert 0.5 < torch.linalg.svdvals(step)[: min(step.shape)].max().item() < 1.3
