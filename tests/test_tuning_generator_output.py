"""CPU: how the gradient of a loss from logits passes a Generator's output -- the mark that lets GeneratorFn leave its log-softmax out holds for exactly
the tensor it was set on, and what watches or changes the gradient on its way is seen."""
import pytest
import torch


class Producer(torch.autograd.Function):
    """stands for GeneratorFn: notes whether the gradient that arrives is marked"""
    seen = []

    @staticmethod
    def forward(ctx, x):
        return x * 2.0

    @staticmethod
    def backward(ctx, d):
        from bmt_amd import ops
        Producer.seen.append(ops._rows_sum_to_zero(d))
        return d * 2.0


def logits_of(pred):
    from bmt_amd import ops
    return ops.GenLogitsFn.apply(pred)


@pytest.mark.parametrize("change,marked", [("none", True), ("look", True), ("scale", False), ("write", False), ("second_consumer", False), ("two_losses", False), ("retain_grad", True)])
def test_the_mark_holds_for_an_untouched_gradient_alone(change, marked):
    Producer.seen.clear()
    x = torch.randn(3, 5).requires_grad_(True)
    pred = Producer.apply(x)
    seen = []
    if change == "look":
        pred.register_hook(lambda g: seen.append(g.clone()))
    elif change == "scale":
        pred.register_hook(lambda g: g * 3.0)
    elif change == "write":
        pred.register_hook(lambda g: g.add_(1.0))
    elif change == "retain_grad":
        pred.retain_grad()
    up = torch.randn(3, 5)
    total = (logits_of(pred) * up).sum()
    want = 2.0 * up
    if change == "scale":
        want = 3.0 * want
    elif change == "write":
        want = want + 2.0
    elif change == "second_consumer":
        total = total + (pred * 7.0).sum()
        want = want + 14.0
    elif change == "two_losses":
        total = total + (logits_of(pred) * up).sum()
        want = 2.0 * want
    total.backward()
    assert Producer.seen == [marked]
    assert torch.allclose(x.grad, want, rtol=1e-6)
    if change == "look":
        assert len(seen) == 1 and torch.equal(seen[0], up)
    if change == "retain_grad":
        assert torch.equal(pred.grad, up)


def test_the_output_itself_has_a_gradient():
    x = torch.randn(3, 5).requires_grad_(True)
    pred = Producer.apply(x)
    up = torch.randn(3, 5)
    (d,) = torch.autograd.grad((logits_of(pred) * up).sum(), pred)
    assert torch.equal(d, up)


def test_values_are_the_output_s_and_written_outputs_are_noticed():
    x = torch.randn(3, 5).requires_grad_(True)
    pred = Producer.apply(x)
    y = logits_of(pred)
    assert torch.equal(y, pred) and y.data_ptr() == pred.data_ptr()
    loss = (y * y).sum()
    with torch.no_grad():
        pred.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
