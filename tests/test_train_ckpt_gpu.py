"""The training pass with 8-bit activation checkpoints (DIONPQGO.activation_checkpoint) and the codeword lookup in the modules
that call it: gradients against the formulas at the kept values, against differences, and against the same step without
checkpoints; what autograd holds; restarts; index dumps back to features."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F64 = torch.float64
U_BF16, U_F32 = 2.0 ** -8, 2.0 ** -24      # half a step, relative: bf16, fp32


def saved_bytes(fn):
    """(result of fn, bytes of the tensors that autograd packed meanwhile, each storage once)."""
    seen = {}

    def pack(t):
        s = t.untyped_storage()
        seen[s.data_ptr()] = s.nbytes()
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        out = fn()
    return out, sum(seen.values())


@pytest.mark.parametrize("keep", ["int8", "e4m3"])
@pytest.mark.parametrize("n,c,d", [(200, 128, 256), (3000, 384, 1024), (333, 128, 384)])
def test_head_gradients_are_the_formula_at_the_kept_values(n, c, d, keep, pkg, native, dev):
    """dW and db of the expansion head from its checkpoint, in fp64 on the host from the same kept values and the bf16 operands
    that the products read.  Bounds: n u for a sum of n terms in fp32 (doubled, the matrix cores may cut); the gradient through
    the second branch is rounded to bf16 once on its way (and summed in fp32 before)."""
    g0 = torch.Generator().manual_seed(3)
    rows = torch.randn(n, c, generator=g0).to(dev)
    par = [torch.randn(*s, generator=g0).mul_(0.05).to(dev).requires_grad_(True) for s in ((d, c, 1, 1), (d,), (c, c, 1, 1), (c,), (d, c, 1, 1), (d,))]
    g = torch.randn(n, d, generator=g0).mul_(1e-3).to(dev)
    head = pkg.pqgo._HeadFunction
    plain = torch.autograd.grad(head.apply(rows, *par, "none"), par, g)
    code, held = saved_bytes(lambda: head.apply(rows, *par, keep))
    _, held_plain = saved_bytes(lambda: head.apply(rows, *par, "none"))
    assert held - held_plain == n * (2 * c + 2 * c // 32) - n * 2 * c * 2
    got = torch.autograd.grad(code, par, g)
    # the operands, rounded as the passes round them
    fh = torch.empty(n, 2 * c, dtype=torch.bfloat16, device=dev)
    fh[:, :c] = rows
    w1, b1, w2a, b2a, w2b, b2b = [p.detach() for p in par]
    w_cat = torch.cat((w1.reshape(d, c), w2b.reshape(d, c)), 1).to(torch.bfloat16).contiguous()
    assert torch.equal(native.expand_head(fh, w2a.reshape(c, c).to(torch.bfloat16).contiguous(), b2a, w_cat, b1 + b2b, d), code)
    kept = native.ckpt_unpack(native.ckpt_pack(fh, keep, keep_sign=True)).cpu().to(F64)
    f, h = kept[:, :c], kept[:, c:]
    assert torch.equal(h > 0, (fh[:, c:] > 0).cpu())
    gb = g.to(torch.bfloat16).cpu().to(F64)
    w2b64 = w_cat[:, c:].cpu().to(F64)
    dh = (gb @ w2b64) * (h > 0)
    dh_size = (gb.abs() @ w2b64.abs()) * (h > 0)
    dh_err = U_BF16 * dh.abs() + 2 * d * U_F32 * dh_size * (1 + U_BF16)
    want = (gb.t() @ f, gb.sum(0), dh.t() @ f, dh.sum(0), gb.t() @ h, gb.sum(0))
    size = (gb.abs().t() @ f.abs(), gb.abs().sum(0), dh.abs().t() @ f.abs(), dh.abs().sum(0), gb.abs().t() @ h.abs(), gb.abs().sum(0))
    more = (0, 0, dh_err.t() @ f.abs(), dh_err.sum(0), 0, 0)
    for i, (a, w, s, m) in enumerate(zip(got, want, size, more)):
        err = (a.cpu().to(F64).reshape(w.shape) - w).abs()
        assert bool((err <= 2 * n * U_F32 * (s + m) + m).all()), (i, float((err / (s + 1e-300)).max()))
    # and near the gradients from what was not rounded: a kept value is off by less than half a step (one step where its sign
    # was kept) of a block whose largest value has 64 (int8) steps or more; e4m3: 2^-4 of itself or 2^-10 / 2^-8 of the largest
    for i, (a, w) in enumerate(zip(got, plain)):
        assert float((a - w).norm() / w.norm()) < (0.02 if keep == "int8" else 0.04), i


def test_quantiser_gradients_against_differences(pkg, native, dev):
    """Directional differences, in fp64 on the host, of the surrogate that the straight-through gradient is the gradient of:
    sum g_zq zn(z) + g_vq (beta mse(zn(z), emb) + book mse(B[idx], zn)), at the kept z."""
    torch.manual_seed(5)
    n, p, k, d, beta, book = 400, 3, 32, 32, 0.25, 1.25
    z = torch.randn(n, p * d, device=dev, requires_grad=True)
    books = (torch.randn(p, k, d, device=dev) * 0.2).requires_grad_(True)
    g = torch.randn(n, p * d, device=dev) * 1e-3
    zq, vq, idx = pkg.pqgo._PQStraightThrough.apply(z, books, beta, book, "int8")
    gz, gb = torch.autograd.grad([zq, vq], [z, books], [g, torch.tensor(0.7, device=dev)])
    zk = native.ckpt_unpack(native.ckpt_pack(z.detach(), "int8")).cpu().to(F64)
    b64, g64, i = books.detach().cpu().to(F64), g.cpu().to(F64), idx.cpu()

    def unit(t):
        t = t.reshape(n, p, d)
        return t / t.norm(dim=-1, keepdim=True)

    emb = torch.stack([b64[q][i[q]] for q in range(p)], 1)

    def of_z(t):
        return (unit(t).reshape(n, -1) * g64).sum() + 0.7 * beta * ((unit(t) - emb) ** 2).mean(dim=(0, 2)).mean()

    def of_books(b):
        return 0.7 * book * ((torch.stack([b[q][i[q]] for q in range(p)], 1) - unit(zk)) ** 2).mean(dim=(0, 2)).mean()

    for value, at, grad in ((of_z, zk, gz), (of_books, b64, gb)):
        for seed in range(3):
            v = torch.randn(at.shape, generator=torch.Generator().manual_seed(seed), dtype=F64)
            t = 1e-5
            slope = float((value(at + t * v) - value(at - t * v)) / (2 * t))
            mine = float((grad.cpu().to(F64) * v).sum())
            # differences: t^2 and 2^-52 / t relative to the terms, ~1e-9; gradients: 64 u relative to their norms
            room = 64 * U_F32 * float(grad.cpu().to(F64).norm() * v.norm()) + 1e-7 * abs(slope) + 1e-9
            assert abs(slope - mine) <= room, (slope, mine)


def test_lookup_gradient_against_differences_and_formula(pkg, dev):
    """The lookup is linear in the books: a difference along any direction is the gradient's, to rounding."""
    torch.manual_seed(6)
    books = torch.randn(3, 20, 24, device=dev, requires_grad=True)
    idx = torch.randint(-1, 20, (3, 3000), device=dev)
    g = torch.randn(3000, 72, device=dev)
    out = pkg.code_lookup(idx, books, 1.5)
    (grad,) = torch.autograd.grad(out, books, g)
    v = torch.randn_like(books)
    slope = (pkg.code_lookup(idx, v, 1.5).to(F64) * g.to(F64)).sum()
    mine = (grad.to(F64) * v.to(F64)).sum()
    assert abs(float(slope - mine)) <= 200 * U_F32 * float((pkg.code_lookup(idx, v.abs(), 1.5).to(F64) * g.abs().to(F64)).sum())
    half = books.detach().to(torch.bfloat16).requires_grad_(True)
    (grad16,) = torch.autograd.grad(pkg.code_lookup(idx, half, 1.5), half, g.to(torch.bfloat16))
    assert grad16.dtype == torch.bfloat16 and float((grad16.float() - grad).norm() / grad.norm()) < 2 * U_BF16
    # through the gradient once more: d <lookup(B)^T g, v> / d g = lookup(v)
    g2 = g.clone().requires_grad_(True)
    (again,) = torch.autograd.grad(pkg.code_lookup(idx, books, 1.5), books, g2, create_graph=True)
    (back,) = torch.autograd.grad(again, g2, v)
    assert torch.equal(back, pkg.code_lookup(idx, v, 1.5))
    # the same code map twice, and one gradient for all rows (a broadcast)
    total = pkg.code_lookup(idx, books, 1.0).sum() + pkg.code_lookup(idx, books, 2.0).sum()
    (grad,) = torch.autograd.grad(total, books)
    counts = torch.stack([torch.bincount(r[r >= 0], minlength=20) for r in idx]).to(torch.float32)
    assert torch.equal(grad, 3.0 * counts.unsqueeze(-1).expand(3, 20, 24))


def step_of(pkg, dev, keep, **config):
    cfg = pkg.configs.pqgo_config(need_initialized="none", drop_prob=0.0, activation_checkpoint=keep, **config)
    m = pkg.build_model(cfg)
    m.load_state_dict(pkg.synth.synth_pqgo_state(cfg, seed=1234), strict=True)
    m = m.to(dev).train()
    img = pkg.synth.synth_images(4, 64, 64, seed=71).to(dev)
    pos = pkg.synth.synth_images(4, 64, 64, seed=72).to(dev)
    label = pkg.synth.synth_labels(4, 64, 64, cfg["num_classes"], seed=71).to(dev)
    g = torch.Generator().manual_seed(9)
    m.model.stego_loss.replay = (torch.rand(4, 11, 11, 2, generator=g) * 2 - 1, torch.rand(4, 11, 11, 2, generator=g) * 2 - 1,
                                 [torch.tensor([1, 2, 3, 0])] * 5)
    (total, out, _preds, _vq), held = saved_bytes(lambda: m(img=img, aug_img=img, label=label, img_pos=pos, it=0))
    total.backward()
    return m, float(total.detach()), {k: p.grad.clone() for k, p in m.named_parameters() if p.requires_grad}, held


@pytest.mark.parametrize("keep", ["int8", "e4m3"])
def test_training_step_with_checkpoints(keep, pkg, dev):
    """One whole step: the forward's losses are those without checkpoints to the bit, gradients of the head and the codebooks are
    off by no more than what was kept is (int8: a few thousandths; e4m3: up to 2^-4 of single values), the probes', which use
    none, are the same to rounding, and autograd holds less."""
    _, loss0, plain, held0 = step_of(pkg, dev, "none")
    m, loss1, got, held1 = step_of(pkg, dev, keep)
    assert m.model.activation_checkpoint == keep and m.model.vq_blocks[0].activation_checkpoint == keep
    assert abs(loss1 - loss0) <= 1e-6 * abs(loss0)
    assert sorted(plain) == sorted(got)
    for name in plain:
        err = float((got[name] - plain[name]).norm() / plain[name].norm())
        limit = (0.02 if keep == "int8" else 0.05) if "evaluator" not in name else 1e-4
        assert err < limit, (name, err)
    # 256 rows: [f | h] 768 bf16 twice (image and pair) and z 1024 fp32 become 1 + 1/32 bytes a value; emb goes, books (1 MB) come
    rows = 256
    assert held0 - held1 >= rows * (2 * 768 * 2 + 1024 * 4) - rows * (2 * 768 + 1024) * 33 // 32 - (1 << 20) - (1 << 16), (held0, held1)


def test_training_step_with_checkpoints_under_autocast(pkg, dev):
    cfg = pkg.configs.pqgo_config(need_initialized="none", activation_checkpoint="int8")
    m = pkg.build_model(cfg)
    m.load_state_dict(pkg.synth.synth_pqgo_state(cfg, seed=1234), strict=True)
    m = m.to(dev).train()
    img = pkg.synth.synth_images(2, 64, 64, seed=71).to(dev)
    label = pkg.synth.synth_labels(2, 64, 64, cfg["num_classes"], seed=71).to(dev)
    scaler = torch.amp.GradScaler("cuda", init_scale=2048)
    with torch.autocast("cuda", dtype=torch.float16):
        total, _out, _preds, _vq = m(img=img, aug_img=img, label=label, img_pos=img.flip(0), it=0)
    scaler.scale(total).backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in m.parameters() if p.requires_grad)


def test_checkpointed_quantiser_with_restart(pkg, dev):
    """A restart writes the codebook after the forward was recorded; the backward reads the codebook it was recorded with."""
    for restart in (False, True):
        torch.manual_seed(2)
        cb = pkg.pqgo.Codebook(64, 32, normalize="l2", use_restart=restart, need_initialized="none").to(dev).train()
        cb.activation_checkpoint = "int8"
        z = torch.randn(2, 32, 6, 6, device=dev, requires_grad=True)
        before = cb.embedding.weight.detach().clone()
        zq, out, _prob, _idx = cb(z, return_prob=False)
        (zq.square().mean() + out["vq-loss"]).backward()
        grads = (z.grad.clone(), cb.embedding.weight.grad.clone())
        assert torch.equal(before, cb.embedding.weight.detach()) != restart
        if restart:
            assert all(torch.equal(a, b) for a, b in zip(grads, without))
        without = grads


def test_checkpoint_setting_is_validated(pkg):
    with pytest.raises(ValueError, match="activation checkpoint"):
        pkg.build_model(pkg.configs.pqgo_config(activation_checkpoint="int4"))
    m = pkg.build_model(pkg.configs.pqgo_config())
    assert m.model.activation_checkpoint == "none"
    with pytest.raises(ValueError, match="activation checkpoint"):
        m.model.activation_checkpoint = "fp8"
    cfg = pkg.configs.pqgo_config()
    del cfg["model"]["activation_checkpoint"]
    assert pkg.build_model(cfg).model.activation_checkpoint == "none"


def test_indices_back_to_features(pkg, dev, tmp_path):
    """The lookup of the eval forward's indices through the wrapper, one codebook, and an index dump on disk is its codewords to
    the bit, and its quantised map up to that map's own rounding: the forward returns zn + (emb - zn) in fp32, whose difference
    is off by u |emb - zn| and whose sum by u |result|; |zn| <= 1 and |emb| < 1/2 here, so 2 u in all."""
    cfg = pkg.configs.S_CFG
    m = pkg.build_model(cfg)
    m.load_state_dict(pkg.synth.synth_pqgo_state(cfg, seed=1234), strict=True)
    m = m.to(dev).eval()
    img = pkg.synth.synth_images(2, 64, 48, seed=3).to(dev)
    label = pkg.synth.synth_labels(2, 64, 48, cfg["num_classes"], seed=3).to(dev)
    vq = m.model.vq_blocks[0]
    with torch.no_grad():
        _code, quantized, (_s, _parts, z_index), _o = m.model(img=img)
        books = torch.stack([q.embedding.weight.detach() for q in vq.quantizers])
        assert float(books.abs().max()) < 0.5
        codewords = torch.cat([books[p][z_index[p]].permute(0, 3, 1, 2) for p in range(8)], dim=1)
        assert torch.equal(vq.lookup(z_index), codewords)
        assert float((codewords - quantized).abs().max()) <= 2 * U_F32
        assert torch.equal(vq.lookup(z_index.to(torch.int16), scale=2.0), codewords * 2)
        assert torch.equal(vq.quantizers[3].lookup(z_index[3]), codewords[:, 384:512])
    with pkg.CodeIndexDump(str(tmp_path / "d"), vq.num_pq, upsample=False) as dump:
        dump.append(z_index, label)
    want = codewords.permute(0, 2, 3, 1).reshape(-1, 1024)
    assert torch.equal(pkg.read_features(str(tmp_path / "d"), vq), want)
    assert torch.equal(pkg.read_features(str(tmp_path / "d"), vq, 5, 17), want[5:17])
    for bad in (z_index[:5], z_index[0], z_index.reshape(8, -1)):
        with pytest.raises(ValueError):
            vq.lookup(bad)
    # differentiable in training mode: every sub-codebook gets its rows' sums
    vq.train()
    vq.lookup(z_index).sum().backward()
    for p, q in enumerate(vq.quantizers):
        counts = torch.bincount(z_index[p].reshape(-1), minlength=256).to(torch.float32)
        assert torch.equal(q.embedding.weight.grad, counts.unsqueeze(1).expand(256, 128))
