"""8-bit activation checkpoints on the GPU (equss_ckpt_pack / _unpack, equss_gemm_tn_ckpt, equss_pq_st_backward_ckpt) against
their definitions in 64 bits on the host.  Roundings counted in units u = 2^-24, half a step of fp32."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F64, F32 = torch.float64, torch.float32


def keep_values(x, fmt, keep_sign):
    """What a checkpoint of x (fp64 on the host, any width) stands for, by the definition, in fp64: blocks of 32 of a row, the
    smallest k >= -110 with which the largest magnitude, rounded, fits.  NaN for blocks that hold an infinity or a NaN."""
    rows, width = x.shape
    x = torch.nn.functional.pad(x, (0, -width % 32)).reshape(-1, 32)
    lost = ~torch.isfinite(x).all(dim=1, keepdim=True)
    x = torch.where(lost, torch.zeros_like(x), x).numpy()
    limit, tiny = (127.0, 1.0) if fmt == "int8" else (448.0, 2.0 ** -9)

    def nearest(v):
        if fmt == "int8":
            return np.rint(v)
        _, e = np.frexp(v)
        step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
        return np.rint(v / step) * step

    peak = np.abs(x).max(axis=1, keepdims=True)
    _, e = np.frexp(peak)
    k = np.maximum(e - (9 if fmt == "int8" else 11), -110)
    for _ in range(4):
        k = k + (nearest(np.ldexp(peak, -k)) > limit)
    v = np.ldexp(x, -k)
    r = nearest(v)
    if keep_sign:
        r = np.where((r == 0) & (v != 0), np.copysign(tiny, v), r)
    out = torch.from_numpy(np.ldexp(r, k))
    out = torch.where(lost, torch.full_like(out, float("nan")), out)
    return out.reshape(rows, -1)[:, :width]


def same(a, b):
    """Equal numbers, NaN where NaN is."""
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a, 0.0, 1e300, -1e300), torch.nan_to_num(b, 0.0, 1e300, -1e300))


def activations(rows, width, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=g) * torch.exp(torch.randn(width, generator=g))
    return x * torch.exp(torch.randn(rows, 1, generator=g))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 384), (3, 31), (7, 33), (5, 1000), (130, 64), (2, 20000), (1500, 768)])
def test_pack_and_unpack_are_the_definition(rows, width, fmt, dtype, native, dev):
    x = activations(rows, width, rows + width).to(dtype)
    for keep in (False, True):
        kept = native.ckpt_pack(x.to(dev), fmt, keep_sign=keep)
        want = keep_values(x.to(F64), fmt, keep)
        assert kept.fmt == fmt and kept.rows == rows and kept.width == width
        assert kept.codes.element_size() == 1 and kept.codes.shape == (rows, -(-width // 32) * 32)
        assert int(kept.codes.cpu().view(torch.uint8)[:, width:].to(torch.int64).sum()) == 0      # padding codes are zero
        assert same(native.ckpt_unpack(kept).cpu().to(F64), want.to(F32).to(F64))
        assert torch.equal(native.ckpt_unpack(kept, torch.bfloat16).cpu().to(F64), want)      # exact: 7 and 4 bits fit into 8
        assert torch.equal(native.ckpt_unpack(kept, torch.float16).cpu(), want.to(torch.float16))
        # half a step of the format at the block's scale, a whole one of the smallest where the sign was kept
        amax = torch.nn.functional.pad(x.to(F64), (0, -width % 32)).reshape(rows, -1, 32).abs().amax(-1).repeat_interleave(32, 1)[:, :width]
        err = (want - x.to(F64)).abs()
        step = amax / 63.5 if fmt == "int8" else torch.maximum(want.abs() / 8, amax * 2.0 ** -16)
        assert bool((err <= step * (1.0 if keep else 0.5)).all())
        if keep:
            assert torch.equal(want > 0, x > 0) and torch.equal(want < 0, x < 0)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_pack_at_the_ends_of_its_range(fmt, native, dev):
    """Magnitudes on either side of the borders where the scale changes, zero blocks, subnormals, the largest finite numbers,
    infinities and NaN, signed zeros; each in a block of its own."""
    edge = 127.5 if fmt == "int8" else 464.0
    below = float(np.nextafter(np.float32(edge), np.float32(0)))
    above = float(np.nextafter(np.float32(edge), np.float32(1e9)))
    firsts = [0.0, -0.0, edge, below, above, -edge, edge * 2.0 ** 40, below * 2.0 ** -40, 1.0, 2.0 ** -102, 2.0 ** -110, 2.0 ** -120, 1e-45,
              3e38, -3.4028234e38, float("inf"), -float("inf"), float("nan")]
    x = torch.zeros(len(firsts), 64)
    for i, f in enumerate(firsts):
        x[i, 0] = f
        x[i, 1] = 0.013 * (f if np.isfinite(f) else 1.0)
        x[i, 5] = -0.0
        x[i, 7] = 1e-45
    for keep in (False, True):
        kept = native.ckpt_pack(x.to(dev), fmt, keep_sign=keep)
        want = keep_values(x.to(F64), fmt, keep)
        got = native.ckpt_unpack(kept).cpu()
        assert same(got.to(F64), want.to(F32).to(F64))
        lost = torch.tensor([not np.isfinite(f) for f in firsts])
        assert bool(torch.isnan(got[lost, :32]).all()) and not bool(torch.isnan(got[~lost]).any()) and not bool(torch.isnan(got[:, 32:]).any())
        assert bool((kept.scales.cpu()[lost, 0] == 255).all())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_pack_takes_strided_rows_and_columns_of_a_checkpoint_read_alike(fmt, native, dev):
    x = activations(77, 200, 3).to(dev)
    whole = native.ckpt_pack(x[:, :192].contiguous(), fmt)
    for view in (x[:, :192], torch.empty(77, 391, device=dev)[:, 1:193].copy_(x[:, :192]), x[:, :192].t().contiguous().t()):
        kept = native.ckpt_pack(view, fmt)
        assert torch.equal(kept.codes.view(torch.uint8), whole.codes.view(torch.uint8)) and torch.equal(kept.scales, whole.scales)
    rep = native.ckpt_pack(x[:1].expand(9, 200), fmt)             # rows that share memory
    assert torch.equal(native.ckpt_unpack(rep), native.ckpt_unpack(native.ckpt_pack(x[:1], fmt)).expand(9, 200))
    values = native.ckpt_unpack(whole)
    for lo, hi in ((0, 32), (64, 192), (160, 192)):
        part = whole.columns(lo, hi)
        assert part.codes.data_ptr() == whole.codes.data_ptr() + lo and torch.equal(native.ckpt_unpack(part), values[:, lo:hi])
    odd = native.ckpt_pack(x, fmt)
    assert torch.equal(native.ckpt_unpack(odd.columns(96, 200)), native.ckpt_unpack(odd)[:, 96:])
    empty = native.ckpt_pack(x[:0], fmt)
    assert empty.rows == 0 and native.ckpt_unpack(empty).shape == (0, 200)


def whole_numbers(rows, width, fmt, seed, dev, native):
    """A checkpoint whose values are whole numbers of at most 15 (exact in either format) with a different scale from row to row."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-15, 16, (rows, width), generator=g).to(F32) * torch.exp2(torch.randint(0, 3, (rows, 1), generator=g).to(F32))
    return x, native.ckpt_pack(x.to(dev), fmt)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("rows,m,n", [(1, 1, 1), (1, 384, 384), (31, 8, 40), (33, 128, 128), (64, 130, 257), (129, 384, 96), (300, 1, 500),
                                      (257, 500, 1), (1000, 200, 333), (4099, 129, 31), (2500, 1024, 768),
                                      (300, 7, 200), (300, 8, 200), (900, 257, 130), (40, 131, 1000), (8000, 9, 20), (30000, 259, 301)])
def test_weight_gradient_is_exact_on_whole_numbers(rows, m, n, fmt, native, dev):
    """Products and sums of whole numbers below 2^24 are exact in fp32 whatever their order: any difference is an element in the
    wrong place.  With and without the ReLU mask, with and without the bias."""
    g = torch.Generator().manual_seed(rows)
    a = torch.randint(-2, 3, (rows, m), generator=g).to(torch.bfloat16)
    v, kept = whole_numbers(rows, n, fmt, 5, dev, native)
    assert torch.equal(native.ckpt_unpack(kept).cpu(), v)
    assert rows * 2 * 60 < 2 ** 24
    assert torch.equal(native.gemm_tn_ckpt(a.to(dev), kept).cpu(), (a.to(F64).t() @ v.to(F64)).to(F32))
    h = torch.relu(torch.randn(rows, m, generator=g))
    for mask_fmt in ("int8", "e4m3"):
        dw, db = native.gemm_tn_ckpt(a.to(dev), kept, relu=native.ckpt_pack(h.to(dev), mask_fmt, keep_sign=True), want_bias=True)
        am = a.to(F64) * (h > 0)
        assert torch.equal(dw.cpu(), (am.t() @ v.to(F64)).to(F32)) and torch.equal(db.cpu(), am.sum(0).to(F32))


@pytest.mark.parametrize("rows,m,n", [(777, 96, 160), (5000, 300, 70)])
def test_weight_gradient_within_the_bound_of_its_sum(rows, m, n, native, dev):
    """Products of two bf16 are exact in fp32; a sum of `rows` terms in any order is off by at most rows u times the sum of
    magnitudes (taken twice: the matrix cores may cut instead of round).  Equal calls give equal bits; a ReLU's masked places hold
    infinities and NaN in the gradient without effect."""
    g = torch.Generator().manual_seed(1)
    a = torch.randn(rows, m, generator=g).to(torch.bfloat16)
    x = activations(rows, n, 2)
    kept = native.ckpt_pack(x.to(dev), "int8")
    v = native.ckpt_unpack(kept).cpu().to(F64)
    dw, db = native.gemm_tn_ckpt(a.to(dev), kept, want_bias=True)
    want, size = a.to(F64).t() @ v, a.to(F64).abs().t() @ v.abs()
    assert bool(((dw.cpu().to(F64) - want).abs() <= 2 * rows * U * size).all())
    assert bool(((db.cpu().to(F64) - a.to(F64).sum(0)).abs() <= 2 * rows * U * a.to(F64).abs().sum(0)).all())
    again = native.gemm_tn_ckpt(a.to(dev), kept, want_bias=True)
    assert torch.equal(dw, again[0]) and torch.equal(db, again[1])
    h = torch.relu(torch.randn(rows, m, generator=g))
    hk = native.ckpt_pack(h.to(dev), "int8", keep_sign=True)
    clean = native.gemm_tn_ckpt(a.to(dev), kept, relu=hk, want_bias=True)
    bad = a.clone()
    bad[h == 0] = float("nan")
    bad[0, h[0] == 0] = float("inf")
    got = native.gemm_tn_ckpt(bad.to(dev), kept, relu=hk, want_bias=True)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])


def test_weight_gradient_takes_views_and_no_rows(native, dev):
    g = torch.Generator().manual_seed(4)
    big = torch.randint(-2, 3, (500, 300), generator=g).to(torch.bfloat16).to(dev)
    v, kept = whole_numbers(500, 256, "int8", 6, dev, native)
    odd = torch.empty(500, 301, dtype=torch.bfloat16, device=dev)
    odd[:, 1:] = big
    for a in (big[:, 7:135], big[:, 3:10], big.t().contiguous().t()[:, :64], odd[:, 1:], odd[:, 2:160], odd[:, 5:12]):
        for lo, hi in ((0, 256), (64, 128), (224, 256)):
            got = native.gemm_tn_ckpt(a, kept.columns(lo, hi))
            assert torch.equal(got.cpu(), (a.cpu().to(F64).t() @ v[:, lo:hi].to(F64)).to(F32))
    far = torch.zeros(600, 2_000_000, dtype=torch.bfloat16, device=dev)      # rows too far apart for 32-bit offsets
    far[:500, 1_000_001:1_000_131] = big[:, :130]
    got = native.gemm_tn_ckpt(far[:500, 1_000_001:1_000_131], kept, want_bias=True)
    assert torch.equal(got[0].cpu(), (big[:, :130].cpu().to(F64).t() @ v.to(F64)).to(F32)) and torch.equal(got[1].cpu(), big[:, :130].cpu().to(F64).sum(0).to(F32))
    del far
    dw, db = native.gemm_tn_ckpt(big[:0], native.ckpt_pack(torch.zeros(0, 48, device=dev)), want_bias=True)
    assert dw.shape == (300, 48) and not bool(dw.any()) and not bool(db.any())
    # a block of NaN spoils its own columns only
    x = torch.randn(64, 96, device=dev)
    x[10, 40] = float("inf")
    for fmt in ("int8", "e4m3"):
        for a in (big[:64], big[:64, :5]):
            dw = native.gemm_tn_ckpt(a, native.ckpt_pack(x, fmt))
            assert bool(torch.isnan(dw[:, 32:64]).all()) and not bool(torch.isnan(dw[:, :32]).any()) and not bool(torch.isnan(dw[:, 64:]).any())
    # one row whose codes have another unit stride
    row = native.ActCheckpoint(kept.codes[:1].t().repeat(1, 2)[:, :1].t(), kept.scales[:1], 256)
    assert torch.equal(native.ckpt_unpack(row).cpu(), v[:1])


def pq_case(n, num_pq, k, d, fmt, seed, skew=1.0):
    g = torch.Generator().manual_seed(seed)
    z = activations(n, num_pq * d, seed + 1)
    z[n // 2] = 0.0
    books = torch.randn(num_pq, k, d, generator=g) * d ** -0.5
    idx = (torch.rand(num_pq, n, generator=g) ** skew * k).long().clamp_(max=k - 1)
    g_zq = torch.randn(n, num_pq * d, generator=g) * 1e-3
    return z, books, idx, g_zq, torch.tensor(0.7)


def pq_formula(z, books, idx, g_zq, g_vq, beta, book):
    """The gradients in fp64 by autograd of the forward's definition, from the given values of z; and the magnitudes their
    roundings go by."""
    n = z.shape[0]
    num_pq, k, d = books.shape
    z, books = z.to(F64).requires_grad_(True), books.to(F64).requires_grad_(True)
    z3 = z.reshape(n, num_pq, d)
    zn = z3 / z3.norm(dim=-1, keepdim=True).clamp_min(1e-12)
    emb = torch.stack([books[p][idx[p]] for p in range(num_pq)], dim=1)
    vq = sum(book * ((emb[:, p] - zn[:, p].detach()) ** 2).mean() + beta * ((zn[:, p] - emb[:, p].detach()) ** 2).mean() for p in range(num_pq)) / num_pq
    zq = zn + (emb - zn).detach()
    loss = vq * g_vq.to(F64)
    if g_zq is not None:
        loss = loss + (zq.reshape(n, -1) * g_zq.to(F64)).sum()
    gz, gb = torch.autograd.grad(loss, [z, books])
    s = float(g_vq) * 2.0 / (n * d * num_pq)
    with torch.no_grad():
        gn = (g_zq.to(F64).reshape(n, num_pq, d).norm(dim=-1) if g_zq is not None else 0.0) + beta * s * (emb.norm(dim=-1) + 1)
        size_z = (gn / z3.norm(dim=-1).clamp_min(1e-12)).unsqueeze(-1).expand(n, num_pq, d).reshape(n, -1)
        terms = book * s * (zn.abs() + emb.abs())
        size_b = torch.zeros_like(books)
        count = torch.zeros(num_pq, k, 1, dtype=F64)
        for p in range(num_pq):
            size_b[p].index_add_(0, idx[p], terms[:, p])
            count[p, :, 0] = torch.bincount(idx[p], minlength=k)
    return gz, gb, size_z, size_b, count


def check_pq(got, want, what):
    gz, gb, size_z, size_b, count = want
    # g_z: the norm's sum of squares is at most 9 roundings deep, the unit vector 8 u, the inner product 9 more, the
    # factor beta s 4 and the last two operations 2: below 32 u of |g'| / |z|; doubled
    if got[0] is not None:
        assert bool(((got[0].cpu().to(F64) - gz).abs() <= 64 * U * size_z).all()), what
    # g_books: 16 u in a term, and one u for every addition that a term passes
    if got[1] is not None:
        assert bool(((got[1].cpu().to(F64) - gb).abs() <= (count + 16) * U * size_b).all()), what


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("n,num_pq,k,d", [(1, 1, 2, 16), (7, 2, 256, 128), (517, 4, 64, 16), (2048, 3, 33, 64), (2049, 3, 32, 64), (3001, 8, 256, 128),
                                          (5000, 3, 7, 32), (9000, 1, 2500, 16)])
def test_quantiser_backward_from_a_checkpoint_matches_the_formula(n, num_pq, k, d, fmt, native, dev):
    z, books, idx, g_zq, g_vq = pq_case(n, num_pq, k, d, fmt, n)
    kept = native.ckpt_pack(z.to(dev), fmt)
    zk = native.ckpt_unpack(kept).cpu()
    for g in (g_zq, None):
        want = pq_formula(zk, books, idx, g, g_vq, 0.25, 1.5)
        args = (kept, books.to(dev), idx.to(dev), g.to(dev) if g is not None else None, g_vq.to(dev), 0.25, 1.5)
        both = native.pq_st_backward_ckpt(*args)
        check_pq(both, want, (n, num_pq, k, d, fmt, g is not None))
        again = native.pq_st_backward_ckpt(*args)
        assert torch.equal(both[0], again[0]) and torch.equal(both[1], again[1])
        rows_only = native.pq_st_backward_ckpt(*args, want_books=False)
        books_only = native.pq_st_backward_ckpt(*args, want_rows=False)
        assert rows_only[1] is None and torch.equal(rows_only[0], both[0])
        assert books_only[0] is None and torch.equal(books_only[1], both[1])


@pytest.mark.parametrize("n", [900, 6000])
def test_quantiser_backward_with_one_busy_codeword_and_places_without_one(n, native, dev):
    """Every row of sub-space 0 on one codeword (its sum crosses every tile); indices outside the codebook in sub-space 1 are
    codewords of zeros whose rows still get their gradient."""
    num_pq, k, d = 2, 40, 32
    z, books, idx, g_zq, g_vq = pq_case(n, num_pq, k, d, "int8", 9)
    idx[0] = 17
    out = torch.arange(n) % 3 == 0
    idx[1, out] = torch.tensor([-1, k, 10 ** 12])[torch.arange(int(out.sum())) % 3]
    padded = torch.cat((books, torch.zeros(num_pq, 1, d)), dim=1)
    kept = native.ckpt_pack(z.to(dev), "int8")
    want = pq_formula(native.ckpt_unpack(kept).cpu(), padded, torch.where((idx < 0) | (idx >= k), torch.full_like(idx, k), idx), g_zq, g_vq, 0.25, 1.0)
    got = native.pq_st_backward_ckpt(kept, books.to(dev), idx.to(dev), g_zq.to(dev), g_vq.to(dev), 0.25, 1.0)
    check_pq(got, (want[0], want[1][:, :k], want[2], want[3][:, :k], want[4][:, :k]), n)


def test_checkpoint_calls_on_a_side_stream_and_in_a_replayed_graph(native, dev):
    """The three calls of a training step, on another stream than the tensors' own and captured: every replay, with eager calls
    of other sizes between them, gives the eager results."""
    n, num_pq, k, d = 3000, 4, 64, 64
    z, books, idx, g_zq, g_vq = pq_case(n, num_pq, k, d, "int8", 12)
    z, books, idx, g_zq, g_vq = z.to(dev), books.to(dev), idx.to(dev), g_zq.to(dev), g_vq.to(dev)
    a = torch.randn(n, 200, device=dev).to(torch.bfloat16)

    def step():
        kept = native.ckpt_pack(z, "int8", keep_sign=True)
        return (native.ckpt_unpack(kept), *native.gemm_tn_ckpt(a, kept, want_bias=True),
                *native.pq_st_backward_ckpt(kept, books, idx, g_zq, g_vq, 0.25, 1.0))

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        z.mul_(2.0 if i % 2 == 0 else 0.5)
        graph.replay()
        torch.cuda.synchronize()
        eager = [t.clone() for t in step()]
        assert all(torch.equal(x, y) for x, y in zip(held, eager)), i
        native.pq_st_backward_ckpt(native.ckpt_pack(z[:2500]), books, idx[:, :2500], None, g_vq, 0.25, 1.0)
        torch.cuda.synchronize()


def test_offsets_past_32_bits(native, dev):
    """Row buffers of more than 2^31 elements: what the calls do with the last rows of them is what they do with these rows alone."""
    rows, num_pq, d, k, tail = 2_200_000, 8, 128, 64, 1500
    width = num_pq * d
    assert rows * width > 2 ** 31
    x = torch.randn(tail, width, device=dev).to(torch.bfloat16)
    big = torch.zeros(rows, width, dtype=torch.bfloat16, device=dev)
    big[-tail:] = x
    for fmt in ("int8", "e4m3"):
        kept, small = native.ckpt_pack(big, fmt), native.ckpt_pack(x, fmt)
        last = native.ActCheckpoint(kept.codes[-tail:], kept.scales[-tail:], width)
        assert torch.equal(last.codes.view(torch.uint8), small.codes.view(torch.uint8)) and torch.equal(last.scales, small.scales)
        back = native.ckpt_unpack(kept, torch.bfloat16)
        assert torch.equal(back[-tail:], native.ckpt_unpack(small, torch.bfloat16)) and not bool(back[:-tail].any())
        del back
    # weight gradient: whole numbers in the last rows only (NaN-free zeros before), exact whatever the row ranges
    a = torch.zeros(rows, 64, dtype=torch.bfloat16, device=dev)
    a[-tail:] = torch.randint(-2, 3, (tail, 64), device=dev).to(torch.bfloat16)
    big[-tail:] = torch.randint(-15, 16, (tail, width), device=dev).to(torch.bfloat16)
    kept = native.ckpt_pack(big, "int8")
    dw, db = native.gemm_tn_ckpt(a, kept, want_bias=True)
    assert torch.equal(dw.to(F64), a[-tail:].to(F64).t() @ big[-tail:].to(F64)) and torch.equal(db.to(F64), a[-tail:].to(F64).sum(0))
    # lookup and its gradient
    idx = torch.randint(-1, k, (num_pq, rows), device=dev)
    books = torch.randn(num_pq, k, d, device=dev).to(torch.bfloat16)
    assert torch.equal(native.code_lookup(idx, books)[-tail:], native.code_lookup(idx[:, -tail:], books))
    assert torch.equal(native.code_lookup_grad(big, idx, k), native.code_lookup_grad(big[-tail:], idx[:, -tail:], k))
    # quantiser: a row's gradient is its own (no vq loss here); the codebooks' is zero without it
    idx.clamp_(min=0)
    books, zero = books.float(), torch.zeros((), device=dev)
    g = torch.zeros(rows, width, device=dev)
    g[-tail:] = torch.randn(tail, width, device=dev)
    gz, gb = native.pq_st_backward_ckpt(kept, books, idx, g, zero, 0.25, 1.0)
    last = native.ActCheckpoint(kept.codes[-tail:].contiguous(), kept.scales[-tail:].contiguous(), width)
    want, _ = native.pq_st_backward_ckpt(last, books, idx[:, -tail:], g[-tail:], zero, 0.25, 1.0)
    assert torch.equal(gz[-tail:], want) and not bool(gz[:-tail].any()) and not bool(gb.any())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("rows,m,n", [(30011, 1001, 701), (2001, 4001, 2601), (25000, 1024, 800), (56003, 1000, 384), (21011, 2500, 391)])
def test_weight_gradient_is_exact_where_the_work_is_large(rows, m, n, fmt, native, dev):
    """More than 2e10 products, where the tiles of 256 stand in: several row ranges and one, edges inside a tile, the bias with and
    without; shapes that lie badly in them; the same through a mask.  Whole numbers below 2^24, exact in fp32 in any order."""
    g = torch.Generator().manual_seed(rows)
    a = torch.randint(-2, 3, (rows, m), generator=g).to(torch.bfloat16)
    v, kept = whole_numbers(rows, n, fmt, 5, dev, native)
    assert rows * m * n >= 2e10 and rows * 2 * 60 < 2 ** 24
    want, sums = a.float().t() @ v.float(), a.float().sum(0)
    assert torch.equal(native.gemm_tn_ckpt(a.to(dev), kept).cpu(), want)
    dw, db = native.gemm_tn_ckpt(a.to(dev), kept, want_bias=True)
    assert torch.equal(dw.cpu(), want) and torch.equal(db.cpu(), sums)
    h = torch.relu(torch.randn(rows, m, generator=g))
    dw, db = native.gemm_tn_ckpt(a.to(dev), kept, relu=native.ckpt_pack(h.to(dev), fmt, keep_sign=True), want_bias=True)
    am = a.float() * (h > 0)
    assert torch.equal(dw.cpu(), am.t() @ v.float()) and torch.equal(db.cpu(), am.sum(0))


@pytest.mark.parametrize("n,num_pq,k,d,fmt", [(70003, 8, 100, 128, "int8"), (140001, 8, 256, 64, "e4m3")])
def test_quantiser_backward_matches_the_formula_where_the_chip_is_full(n, num_pq, k, d, fmt, native, dev):
    """Enough rows for tiles of 64 everywhere (rows / 64 times sub-spaces times lanes a row, 2^18 or more); bounds as above."""
    assert (n + 63) // 64 * num_pq * (d // 4) >= 2 ** 18
    z, books, idx, g_zq, g_vq = pq_case(n, num_pq, k, d, fmt, n, skew=2.0)
    kept = native.ckpt_pack(z.to(dev), fmt)
    want = pq_formula(native.ckpt_unpack(kept).cpu(), books, idx, g_zq, g_vq, 0.25, 1.5)
    check_pq(native.pq_st_backward_ckpt(kept, books.to(dev), idx.to(dev), g_zq.to(dev), g_vq.to(dev), 0.25, 1.5), want, (n, num_pq, k, d, fmt))
