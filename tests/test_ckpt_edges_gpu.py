"""The checkpointed training pass and its operators where layouts, missing gradients and the ends of the number formats meet
them."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F64 = torch.float64
U = 2.0 ** -24


@pytest.mark.parametrize("keep", ["none", "int8", "e4m3"])
def test_head_gradients_of_one_image_whose_gradient_lies_by_channels(keep, pkg, dev):
    """With one image, the rows of an NCHW-contiguous gradient have a column stride of h w and a row stride of 1.  Whole numbers
    of at most 256 throughout (sums below 2^24): every product and sum is exact, so both layouts give equal bits."""
    h, w, c, d = 9, 7, 128, 256
    g0 = torch.Generator().manual_seed(11)

    def whole(*shape):
        return torch.randint(-1, 2, shape, generator=g0).float().to(dev)

    rows = whole(h * w, c)
    par = [whole(*s).requires_grad_(True) for s in ((d, c, 1, 1), (d,), (c, c, 1, 1), (c,), (d, c, 1, 1), (d,))]
    grad = whole(1, d, h, w)
    by_rows = grad.permute(0, 2, 3, 1).reshape(-1, d).contiguous()
    by_channels = grad.permute(0, 2, 3, 1).reshape(-1, d)
    assert by_channels.stride() == (1, h * w) and torch.equal(by_rows, by_channels)
    code = pkg.pqgo._HeadFunction.apply(rows, *par, keep)
    want = torch.autograd.grad(code, par, by_rows, retain_graph=True)
    got = torch.autograd.grad(code, par, by_channels)
    assert all(bool(t.any()) for t in want) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_row_products_take_operands_of_any_strides(native, dev):
    """native.gemm_bf16 of transposed, column-strided and one-row operands; an output it cannot write is refused."""
    g = torch.Generator().manual_seed(12)
    a = torch.randint(-2, 3, (256, 128), generator=g).to(torch.bfloat16).to(dev)
    w = torch.randint(-2, 3, (128, 128), generator=g).to(torch.bfloat16).to(dev)
    want = (a.cpu().to(F64) @ w.cpu().to(F64).t()).to(torch.bfloat16)
    for x in (a, a.t().contiguous().t(), a.repeat_interleave(2, dim=1)[:, ::2]):
        for y in (w, w.t().contiguous().t(), w.repeat_interleave(2, dim=1)[:, ::2]):
            assert torch.equal(native.gemm_bf16(x, y, None, native.EPI_BF16).cpu(), want)
    one = a.t().contiguous().t()[:1]
    assert torch.equal(native.gemm_bf16(one, w, None, native.EPI_BF16).cpu(), want[:1])
    with pytest.raises(ValueError, match="out"):
        native.gemm_bf16(a, w, None, native.EPI_BF16, out=torch.empty(128, 256, dtype=torch.bfloat16, device=dev).t())


@pytest.mark.parametrize("keep", ["none", "int8", "e4m3"])
def test_training_step_of_one_image(keep, pkg, dev):
    cfg = pkg.configs.pqgo_config(need_initialized="none", drop_prob=0.0, activation_checkpoint=keep)
    m = pkg.build_model(cfg)
    m.load_state_dict(pkg.synth.synth_pqgo_state(cfg, seed=1234), strict=True)
    m = m.to(dev).train()
    img = pkg.synth.synth_images(1, 64, 64, seed=71).to(dev)
    label = pkg.synth.synth_labels(1, 64, 64, cfg["num_classes"], seed=71).to(dev)
    total, _out, _preds, _vq = m(img=img, aug_img=img, label=label, img_pos=img.flip(3), it=0)
    total.backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in m.parameters() if p.requires_grad)


@pytest.mark.parametrize("keep", ["none", "int8"])
@pytest.mark.parametrize("closed_form", [False, True])
def test_quantiser_gradient_of_the_quantised_output_alone(closed_form, keep, pkg, native, dev, monkeypatch):
    """A loss that reaches the quantiser through zq only, and one through vq only, in every branch of the backward, against the
    formula in fp64: g_z = (g - zn <zn, g>) / |z| at the z that the branch keeps (64 u of |g| / |z|: the norm's sum, two products
    and the projection are below 32 roundings deep)."""
    monkeypatch.setattr(pkg.pqgo._PQStraightThrough, "hip_backward", not closed_form)
    torch.manual_seed(7)
    n, p, k, d = 300, 2, 32, 32
    z = torch.randn(n, p * d, device=dev, requires_grad=True)
    books = (torch.randn(p, k, d, device=dev) * 0.2).requires_grad_(True)
    g = torch.randn(n, p * d, device=dev)
    zq, vq, _ = pkg.pqgo._PQStraightThrough.apply(z, books, 0.25, 1.0, keep)
    gz, gb = torch.autograd.grad(zq, [z, books], g, retain_graph=True)
    zk = z.detach() if keep == "none" else native.ckpt_unpack(native.ckpt_pack(z.detach(), keep))
    z3, g3 = zk.cpu().to(F64).reshape(n, p, d), g.cpu().to(F64).reshape(n, p, d)
    norm = z3.norm(dim=-1, keepdim=True)
    zn = z3 / norm
    want = (g3 - zn * (zn * g3).sum(-1, keepdim=True)) / norm
    assert bool(((gz.cpu().to(F64).reshape(n, p, d) - want).abs() <= 64 * U * g3.norm(dim=-1, keepdim=True) / norm).all())
    assert not bool(gb.any())
    gz, gb = torch.autograd.grad(vq, [z, books])
    assert bool(gz.any()) and bool(gb.any())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_mask_of_a_block_that_holds_an_infinity_or_a_nan(fmt, native, dev):
    """Signs are kept there too: a place counts where its value is positive, an infinity among them, and the block still reads
    back as NaN throughout.  What lies outside such blocks is not touched."""
    g = torch.Generator().manual_seed(13)
    rows, m, n = 40, 96, 64
    h = torch.randn(rows, m, generator=g)
    h[3, 5], h[7, 40], h[9, 70], h[11, 71] = float("inf"), -float("inf"), float("nan"), float("inf")
    h[3, 6] = 0.0
    h[11, 64:71] = torch.tensor([1e-45, -1e-45, 0.0, -0.0, 3e38, -3e38, float("nan")])
    kept = native.ckpt_pack(h.to(dev), fmt, keep_sign=True)
    codes = kept.codes.view(torch.int8).cpu()
    assert torch.equal(codes > 0, h > 0) and torch.equal(codes < 0, h < 0)
    lost = (~torch.isfinite(h)).reshape(rows, -1, 32).any(-1).repeat_interleave(32, 1)
    assert bool((kept.scales.cpu()[lost[:, ::32]] == 255).all())
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        back = native.ckpt_unpack(kept, dtype).cpu()
        assert bool(torch.isnan(back[lost]).all()) and not bool(torch.isnan(back[~lost]).any())
    a = torch.randint(-2, 3, (rows, m), generator=g).to(torch.bfloat16)
    v = torch.randint(-15, 16, (rows, n), generator=g).float()
    am = a.to(F64) * (h > 0)
    vk = native.ckpt_pack(v.to(dev), fmt)
    dw, db = native.gemm_tn_ckpt(a.to(dev), vk, relu=kept, want_bias=True)
    assert torch.equal(dw.cpu(), (am.t() @ v.to(F64)).float()) and torch.equal(db.cpu(), am.sum(0).float())
    dw = native.gemm_tn_ckpt(a[:, :5].to(dev), vk, relu=native.ckpt_pack(h[:, :5].to(dev), fmt, keep_sign=True))     # narrow form
    assert torch.equal(dw.cpu(), (am[:, :5].t() @ v.to(F64)).float())
    # as the kept input of the layer: its columns of the product are not finite, the others are
    spoilt = native.gemm_tn_ckpt(torch.ones(rows, 16, dtype=torch.bfloat16, device=dev), kept).cpu()
    cols = lost.any(0)
    assert not bool(torch.isfinite(spoilt[:, cols]).any()) and bool(torch.isfinite(spoilt[:, ~cols]).all())


def test_quantiser_backward_shows_a_lost_block_throughout_its_codeword(native, dev):
    """A block that lost its values spoils its sub-space of its row and the codeword's gradient, all d columns, nothing else."""
    n, p, k, d = 50, 2, 8, 64
    z = torch.randn(n, p * d, generator=torch.Generator().manual_seed(14))
    z[20, 70] = float("inf")
    books, idx = torch.randn(p, k, d), torch.arange(n).remainder(k).repeat(p, 1)
    for keep in (False, True):
        for fmt in ("int8", "e4m3"):
            kept = native.ckpt_pack(z.to(dev), fmt, keep_sign=keep)
            gz, gb = native.pq_st_backward_ckpt(kept, books.to(dev), idx.to(dev), torch.randn(n, p * d, device=dev), torch.ones((), device=dev), 0.25, 1.0)
            bad_z, bad_b = torch.isnan(gz).cpu(), torch.isnan(gb).cpu()
            assert bool(bad_z[20, d:].all()) and int(bad_z.sum()) == d
            assert bool(bad_b[1, 20 % k].all()) and int(bad_b.sum()) == d


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_largest_numbers_of_every_type(fmt, native, dev):
    """A block's largest number decides the scale 2^k: int8 keeps 127 2^(k) up to 127.5 2^k and takes k + 1 from there, e4m3 448 up
    to 464.  With the raised scale 63.5 (int8) or 248 (e4m3) and more of it round to 64 or 256, i.e. to 2^128 at the top of fp32
    and bf16 and to 2^16 at the top of fp16; everything below stays finite and within half a step."""
    raised, up, step = (127.5 / 128, 63.5 / 64, 1 / 64) if fmt == "int8" else (464 / 512, 248 / 256, 16 / 256)
    for dtype, top in ((torch.float32, 128), (torch.bfloat16, 128), (torch.float16, 16)):
        largest = torch.finfo(dtype).max
        x = torch.zeros(6, 32, dtype=F64)
        x[:, 0] = torch.tensor([largest, -largest, raised * 0.995 * 2.0 ** top, up * 0.95 * 2.0 ** top, largest, largest])
        x[4, 1], x[5, 1] = -up * 2.0 ** top, up * 0.96 * 2.0 ** top
        x = x.to(dtype)
        back = {t: native.ckpt_unpack(native.ckpt_pack(x.to(dev), fmt), t).cpu().to(F64) for t in (torch.float32, torch.bfloat16, torch.float16)}
        inf = float("inf")
        for t in (torch.float32, torch.bfloat16):
            value = 2.0 ** top if top < 128 else inf
            assert back[t][0, 0] == value and back[t][1, 0] == -value and back[t][4, 1] == -value
        if top == 16:
            got = back[torch.float16]
            assert got[0, 0] == inf and got[1, 0] == -inf and got[4, 1] == -inf
        finite = back[dtype]
        for r, c in ((2, 0), (3, 0), (5, 1)):
            assert abs(float(finite[r, c] - x[r, c].to(F64))) <= step / 2 * 2.0 ** top, (dtype, r)
        assert bool((finite[:, 2:] == 0).all())                       # zeros beside them stay zeros: no NaN


@pytest.mark.parametrize("branch", ["none", "closed form", "int8", "e4m3"])
def test_quantiser_gradient_where_the_norm_is_clamped(branch, pkg, native, dev, monkeypatch):
    """0 < |z| < 1e-12: the norm is the constant 1e-12 there and its derivative zero, so nothing is projected out, as autograd has
    it through clamp_min in fp64.  A dozen roundings at most on the terms' magnitudes, 64 u where the norm is the row's own."""
    monkeypatch.setattr(pkg.pqgo._PQStraightThrough, "hip_backward", branch != "closed form")
    keep = branch if branch in ("int8", "e4m3") else "none"
    torch.manual_seed(15)
    n, p, k, d, beta, book = 120, 2, 32, 32, 0.25, 1.0
    z = torch.randn(n, p, d) * torch.tensor([1.0, 1e-13, 3e-14, 1e-16])[torch.arange(n) % 4].reshape(n, 1, 1)
    z = z.reshape(n, p * d).to(dev).requires_grad_(True)
    books = (torch.randn(p, k, d, device=dev) * 0.2).requires_grad_(True)
    g = torch.randn(n, p * d, device=dev)
    zq, vq, idx = pkg.pqgo._PQStraightThrough.apply(z, books, beta, book, keep)
    gz, gb = torch.autograd.grad([zq, vq], [z, books], [g, torch.tensor(300.0, device=dev)])
    zk = z.detach() if keep == "none" else native.ckpt_unpack(native.ckpt_pack(z.detach(), keep))
    z64, b64, i = zk.cpu().to(F64).requires_grad_(True), books.detach().cpu().to(F64).requires_grad_(True), idx.cpu()
    z3 = z64.reshape(n, p, d)
    norm = z3.norm(dim=-1, keepdim=True).clamp_min(1e-12)
    zn, emb = z3 / norm, torch.stack([b64[q][i[q]] for q in range(p)], 1)
    loss = 300.0 * (beta * ((zn - emb.detach()) ** 2).mean() + book * ((emb - zn.detach()) ** 2).mean()) + (zn.reshape(n, -1) * g.cpu().to(F64)).sum()
    want_z, want_b = torch.autograd.grad(loss, [z64, b64])
    s = 300.0 * 2 / (n * p * d)
    size = (g.cpu().to(F64).reshape(n, p, d).norm(dim=-1, keepdim=True) + beta * s * (emb.norm(dim=-1, keepdim=True) + 1)) / norm
    assert bool((norm[torch.arange(n) % 4 != 0] == 1e-12).all())
    assert bool(((gz.cpu().to(F64) - want_z).abs().reshape(n, p, d) <= 64 * U * size).all())
    terms = (book * s * (zn.abs() + emb.abs())).detach()
    for q in range(p):
        room, count = torch.zeros(k, d, dtype=F64).index_add_(0, i[q], terms[:, q]), torch.bincount(i[q], minlength=k).to(F64).unsqueeze(1)
        assert bool(((gb[q].cpu().to(F64) - want_b[q]).abs() <= (count + 16) * U * room).all())
