"""GPU: the 8-bit operators beside PyTorch's autograd: what they write to counts as written."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def layer(ops, cuda):
    return ops.Int8Linear(torch.randn(40, 64, device="cuda"))


def writes(ops, layer):
    """(tensor that is written, the call) of every call that writes to a tensor of the caller's."""
    x = torch.randn(20, 64, device="cuda")
    codes, scales = ops.quantize_rows(x)
    for make in (lambda: torch.zeros(20, 40, device="cuda"),):
        yield make(), lambda t: layer.forward(x, out=t)
        yield make(), lambda t: layer.forward(x, out=t, accumulate=True)
        yield make(), lambda t: layer.forward_codes(codes, scales, out=t)
        yield make(), lambda t: layer.forward_codes(codes, scales, out=t, accumulate=True)
    yield x.clone(), lambda t: ops.norm_block(t, x, in_place=True)
    yield x.clone(), lambda t: ops.norm_block(t, x, out_dtype=torch.float32, in_place=True)


def test_a_saved_tensor_that_was_written_to_is_noticed(ops, cuda, layer):
    for t, call in writes(ops, layer):
        w = torch.ones_like(t, requires_grad=True)
        loss = (w * t).sum()                   # saves t for w's gradient
        call(t)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_a_tensor_that_requires_a_gradient_is_not_written_to(ops, cuda, layer):
    for t, call in writes(ops, layer):
        before = t.clone()
        t.requires_grad_()
        with pytest.raises(ops.InvalidArgument, match="gradient"):
            call(t)
        assert torch.equal(t, before)
        with torch.no_grad():
            call(t)
        assert not torch.equal(t, before)


def test_inference_mode_and_inputs_that_are_only_read(ops, cuda, layer):
    with torch.inference_mode():
        for t, call in writes(ops, layer):
            call(t)
    x = torch.randn(20, 64, device="cuda")
    ops.norm_block(x, x, out_dtype=torch.float32)
    layer.forward(x)
    ops.quantize_rows(x)
    assert x._version == 0
    assert not layer.forward(x.clone().requires_grad_()).requires_grad
