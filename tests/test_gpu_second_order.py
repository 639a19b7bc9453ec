"""The token operators' gradients are once differentiable: a second derivative through them is refused
with an error, not left out of the result (it would be, silently, where another path through the
graph has one)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def calls(gen):
    from ttsplat.attention import attention
    from ttsplat.embedding import embedding
    from ttsplat.norm import layer_norm

    def leaf(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).requires_grad_(True)
    q, k, v = leaf(1, 2, 5, 8), leaf(1, 2, 7, 8), leaf(1, 2, 7, 8)
    x, w, table = leaf(6, 8), leaf(8), leaf(9, 8)
    ids = torch.arange(9, device="cuda")
    return {"attention": (lambda: attention(q, k, v), q), "norm": (lambda: layer_norm(x, w), x),
            "embedding": (lambda: embedding(table, ids), table)}


@pytest.mark.parametrize("name", ["attention", "norm", "embedding"])
def test_second_derivative_refused(name):
    run, leaf = calls(torch.Generator(device="cuda").manual_seed(3))[name]
    y = run()
    (plain,) = torch.autograd.grad(y.square().sum(), leaf)
    # the square of the leaf has a second derivative of its own
    (g,) = torch.autograd.grad(run().square().sum() + leaf.square().sum(), leaf, create_graph=True)
    assert torch.equal(g, plain + 2 * leaf)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(g.sum(), leaf, retain_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()
