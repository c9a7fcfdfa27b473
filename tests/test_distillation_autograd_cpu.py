"""The distillation functions under autograd: differentiable once, said so where it is asked for twice. (No GPU: the kernels are
replaced by a loss sum z^2 and its gradient.)"""
import pytest
import torch

from uno_amd import kernels as K, objectives
from uno_amd.objectives import top_k_distillation_loss
from uno_amd.training.losses import token_normalized_top_k_distillation


class _Head:
    weight = torch.randn(8, 4)
    weight_t = weight.t().contiguous()


@pytest.fixture(autouse=True)
def plain(monkeypatch):
    monkeypatch.setattr(objectives, "_distill_fwd", lambda z, *a: ((z.detach() ** 2).sum(), torch.zeros(z.shape[0], 2)))

    def bwd(z, values, indices, stat, g, inv_n, scale, tau, grad):
        with torch.no_grad():
            grad.copy_(2 * z * g)
        return grad.detach()
    monkeypatch.setattr(objectives, "_distill_bwd", bwd)
    monkeypatch.setattr(K, "gemm_nt", lambda a, b: (a @ b.t()).detach())


def _logits_loss(x):
    return token_normalized_top_k_distillation(x, torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64), 3)


def _head_loss(x):
    return top_k_distillation_loss(_Head, x, torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64), torch.ones(1))


LOSSES = {"logits": (_logits_loss, 8), "head": (_head_loss, 4)}


@pytest.mark.parametrize("name", LOSSES)
def test_once(name):
    loss, width = LOSSES[name]
    x = torch.randn(3, width, requires_grad=True)
    loss(x).backward()
    ref = 2 * x.detach() if name == "logits" else 2 * x.detach() @ _Head.weight.t() @ _Head.weight
    torch.testing.assert_close(x.grad, ref)


@pytest.mark.parametrize("name", LOSSES)
def test_a_second_derivative_is_refused(name):
    """Beside a term that has one, whose part alone would come back."""
    loss, width = LOSSES[name]
    x = torch.randn(3, width, requires_grad=True)
    (grad,) = torch.autograd.grad(loss(x) + (x ** 3).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        (grad ** 2).sum().backward()


def test_a_second_backward():
    """Over given logits it repeats the first; over the LM head, whose logits the first one overwrites, it is refused."""
    x = torch.randn(3, 8, requires_grad=True)
    out = _logits_loss(x)
    first = torch.autograd.grad(out, x, retain_graph=True)[0]
    assert torch.equal(first, torch.autograd.grad(out, x)[0])
    x = torch.randn(3, 4, requires_grad=True)
    out = _head_loss(x)
    torch.autograd.grad(out, x, retain_graph=True)
    with pytest.raises(RuntimeError, match="a second time"):
        torch.autograd.grad(out, x)
