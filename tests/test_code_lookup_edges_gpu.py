"""The codeword lookup and its gradient at the sizes and uses that their variants part at, and forward-mode differentiation."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu

F64 = torch.float64
U = 2.0 ** -24


def test_lookup_carries_tangents(pkg, dev):
    """The lookup is linear in the books: its tangent is the lookup of the tangent, and its gradient's tangent the gradient of
    the tangent."""
    torch.manual_seed(21)
    books, t = torch.randn(3, 20, 24, device=dev), torch.randn(3, 20, 24, device=dev)
    idx = torch.randint(-1, 21, (3, 500), device=dev)
    with fwd.dual_level():
        out, tangent = fwd.unpack_dual(pkg.code_lookup(idx, fwd.make_dual(books, t), 1.5))
        assert torch.equal(out, pkg.code_lookup(idx, books, 1.5)) and torch.equal(tangent, pkg.code_lookup(idx, t, 1.5))
    # forward over reverse: d/ds of the gradient of <lookup(B)^2, 1> at B + s t is 2 lookup^T lookup t
    with fwd.dual_level():
        dual = fwd.make_dual(books.clone().requires_grad_(True), t)
        (grad,) = torch.autograd.grad(pkg.code_lookup(idx, dual, 1.0).square().sum(), dual, create_graph=True)
        tangent = fwd.unpack_dual(grad).tangent
    counts = torch.stack([torch.bincount(r[(r >= 0) & (r < 20)], minlength=20) for r in idx]).float().unsqueeze(-1)
    # (a product with a whole number by repeated addition: at most count additions of u each)
    assert bool(((tangent - 2 * counts * t).abs() <= (counts + 2) * U * (2 * counts * t).abs()).all())


@pytest.mark.parametrize("normalize", ["z_norm", "none"])
def test_training_quantiser_carries_tangents(normalize, pkg, dev):
    """The quantiser's z_norm / none training branch with a dual codebook: the vq loss's tangent is its directional difference."""
    torch.manual_seed(22)
    p, k, d, n = 1, 32, 32, 200
    rows = torch.randn(n, d, device=dev)
    books, t = torch.randn(p, k, d, device=dev), torch.randn(p, k, d, device=dev)

    def loss(b):
        return pkg.pqgo._quantize_rows(rows, b, normalize, 0.25, 1.0, True, None)[2]["vq-loss"]

    with fwd.dual_level():
        tangent = fwd.unpack_dual(loss(fwd.make_dual(books.clone().requires_grad_(True), t))).tangent
    b = books.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(loss(b), b)
    # both are sums of n d products in fp32, in different orders: n d u of the magnitudes' sum at most
    assert abs(float((grad.to(F64) * t.to(F64)).sum() - tangent.detach().to(F64))) <= n * d * U * float((grad.abs().to(F64) * t.abs().to(F64)).sum())


def test_vector_quantizer_carries_tangents(pkg, dev):
    torch.manual_seed(23)
    vq = pkg.quantizer.VectorQuantizer(num_codebook=32, embed_dim=32, normalize="none").to(dev).train()
    z, t = torch.randn(2, 32, 5, 5, device=dev), torch.randn(32, 32, device=dev)
    (grad,) = torch.autograd.grad(vq(z)[1]["loss"], vq.codebook.weight)
    weight = vq.codebook.weight.detach().clone()
    del vq.codebook.weight
    with fwd.dual_level():
        vq.codebook.weight = fwd.make_dual(weight.requires_grad_(True), t)
        tangent = fwd.unpack_dual(vq(z)[1]["loss"]).tangent
    assert abs(float((grad.to(F64) * t.to(F64)).sum() - tangent.detach().to(F64))) <= 1600 * U * float((grad.abs().to(F64) * t.abs().to(F64)).sum())
