"""What the operators' autograd nodes keep for the backward pass: changed in
place before it, it is an error and not another gradient."""
import pytest
import torch

import garfield_amd as gf

pytestmark = pytest.mark.gpu


def _rows(made):
    g = torch.Generator().manual_seed(3)
    w = gf.mx_quantise(torch.randn(30, 96, generator=g).cuda())
    if made == "split":
        w.codes
    elif made == "own":
        w = gf.MXRows(w.codes.clone(), w.scales.clone(), 96)
    elif made == "slice":
        w = gf.MXRows(w.codes.clone(), w.scales.clone(), 96)[4:20]
    return w


@pytest.mark.parametrize("made", ["quantised", "split", "own", "slice"])
@pytest.mark.parametrize("part", ["codes", "scales"])
def test_rows_changed_before_the_backward_pass(made, part):
    print("case saved rows", made, part, flush=True)
    w = _rows(made)
    x = torch.randn(5, 96, device="cuda", requires_grad=True)
    y = gf.mx_product(x, w)
    want = gf.mx_product_grad(torch.ones_like(y), w)
    (d,) = torch.autograd.grad(y.sum(), x, retain_graph=True)
    assert torch.equal(d, want)
    getattr(w, part)[3].zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    # a new product takes the rows as they are now
    (d,) = torch.autograd.grad(gf.mx_product(x, w).sum(), x)
    assert torch.equal(d, gf.mx_product_grad(torch.ones_like(y), w)) and not torch.equal(d, want)


def test_rows_of_inference_mode_and_repeated_passes():
    """Frozen rows made in inference mode train what stands in front of them; a
    product alone can be gone back through twice."""
    print("case inference rows", flush=True)
    with torch.inference_mode():
        w = _rows("quantised")
    x = torch.randn(5, 96, device="cuda", requires_grad=True)
    y = gf.mx_product(x, w).sum()
    y.backward()
    first = x.grad.clone()
    y.backward()
    assert torch.equal(first, gf.mx_product_grad(torch.ones(5, 30, device="cuda"), w))
    assert torch.equal(x.grad, 2 * first)


def test_no_gradient_through_what_is_not_rows():
    x = torch.randn(5, 96, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="MXRows"):
        gf.mx_product(x, x)
