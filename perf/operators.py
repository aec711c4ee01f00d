"""Cases by which the operators of the 8-bit training pass and of the codeword lookup are measured.

Five operators, each with a plain form (elementary torch operations in 32 bits) and the framework's own call:

  pack         an activation kept in 8 bits between forward and backward and read back: native.ckpt_pack, native.ckpt_unpack
  wgrad        weight and bias gradient of a linear layer whose input was kept that way: native.gemm_tn_ckpt
  pq           backward of the product quantisation whose input was kept that way: native.pq_st_backward_ckpt
  lookup       codewords gathered by their indices, with a scale: native.code_lookup
  lookup_grad  its gradient, summed by sorted codes: native.code_lookup_grad

The 8-bit form: blocks of 32 consecutive channels of a row share a scale 2^k, k the smallest integer, at least -110, with which
the block's largest magnitude does not pass the format's largest value (int8: 127, e4m3: 448) after rounding; values are rounded to
nearest even.  "keep": a value other than zero that would round to zero takes the smallest magnitude of its sign instead, so that
the mask of a ReLU survives.  `own` is set from outside: False runs the plain forms, True the framework's kernels."""
import math

import torch

own = False

BLOCK = 32
KMIN = -110
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
INTS = {"int64": torch.int64, "int32": torch.int32, "int16": torch.int16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2, "int64": 8, "int32": 4, "int16": 2}
# the most a drawn case may have: elements of the row buffer, which is what every operator's time goes by
MOST = 102400 * 1024


def listed():
    return [
        # one pooled token of ViT-S kept and read back: nothing but latency
        {"name": "pack_token", "op": "pack", "rows": 1, "width": 384, "type": "bf16", "fmt": "int8", "keep": True},
        # a ragged batch of rows whose width ends inside a block of 32
        {"name": "pack_ragged", "op": "pack", "rows": 3001, "width": 1000, "type": "fp32", "fmt": "e4m3", "keep": False},
        # [features | ReLU branch] of the expansion head for 64 images of 320 x 320: what the head's backward needs
        {"name": "pack_head", "op": "pack", "rows": 102400, "width": 768, "type": "bf16", "fmt": "int8", "keep": True},
        # the head's first weight gradient for 4 images of 64 x 64
        {"name": "wgrad_small", "op": "wgrad", "rows": 256, "m": 1024, "n": 768, "fmt": "int8", "relu": False},
        # sizes off every tile, through a ReLU: 13 crops of 16 x 61 patches
        {"name": "wgrad_ragged", "op": "wgrad", "rows": 12688, "m": 200, "n": 333, "fmt": "e4m3", "relu": True},
        # [dW1 | dW2b] of the head for 64 images of 320 x 320
        {"name": "wgrad_head", "op": "wgrad", "rows": 102400, "m": 1024, "n": 768, "fmt": "int8", "relu": False},
        # the quantiser of 8 x 256 codewords, 4 images of 64 x 64, a gradient arriving through the quantised output
        {"name": "pq_small", "op": "pq", "rows": 256, "pq": 8, "k": 256, "d": 128, "fmt": "e4m3", "gzq": True},
        # the same quantiser in the training step of 64 images of 320 x 320
        {"name": "pq_step", "op": "pq", "rows": 102400, "pq": 8, "k": 256, "d": 128, "fmt": "int8", "gzq": True},
        # a few tokens' codes turned back into features, some of them padding
        {"name": "lookup_few", "op": "lookup", "rows": 5, "pq": 8, "k": 256, "d": 128, "type": "fp32", "index": "int64", "by_row": False, "scale": 1.0},
        # an index dump (int16, one row a patch) turned back into bf16 features, 64 images of 320 x 320
        {"name": "lookup_dump", "op": "lookup", "rows": 102400, "pq": 8, "k": 256, "d": 128, "type": "bf16", "index": "int16", "by_row": True, "scale": 11.3125},
        # a short batch against a codebook much larger than the batch, narrow codewords
        {"name": "lookup_grad_wide", "op": "lookup_grad", "rows": 3137, "pq": 1, "k": 16384, "d": 16, "type": "bf16", "index": "int32", "by_row": False, "scale": 4.0},
        # the codebooks' gradient in the training step of 64 images of 320 x 320
        {"name": "lookup_grad_step", "op": "lookup_grad", "rows": 102400, "pq": 8, "k": 256, "d": 128, "type": "fp32", "index": "int64", "by_row": False, "scale": 1.0},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["pack", "wgrad", "pq", "lookup", "lookup_grad"])
    rows = _log(rng, 1, 102400)
    fmt = rng.choice(["int8", "e4m3"])
    if op == "pack":
        width = min(_log(rng, 16, 2048), max(16, 102400 * 768 // rows))
        return {"op": op, "rows": rows, "width": width, "type": rng.choice(["fp32", "bf16", "fp16"]) if rows < 60000 else "bf16",
                "fmt": fmt, "keep": rng.random() < 0.5}
    if op == "wgrad":
        # cost: rows * m * n products and rows * (2 m + n) bytes, both below wgrad_head's
        m, n = _log(rng, 32, 1024), _log(rng, 32, 768)
        return {"op": op, "rows": rows, "m": m, "n": n, "fmt": fmt, "relu": rng.random() < 0.5 and rows * m <= 102400 * 512}
    d = rng.choice([16, 32, 64, 128])
    pq = min(_log(rng, 1, 16), max(1, MOST // (rows * d)))
    if op == "pq":
        return {"op": op, "rows": rows, "pq": pq, "k": _log(rng, 2, 512), "d": d, "fmt": fmt, "gzq": rng.random() < 0.6}
    if rng.random() < 0.3:  # widths that no vector load divides
        d = rng.randint(3, 127)
        pq = min(pq, max(1, MOST // (rows * d)))
    k = _log(rng, 2, 16384 if pq <= 2 else 1024)
    return {"op": op, "rows": rows, "pq": pq, "k": k, "d": d, "type": rng.choice(["fp32", "bf16", "fp16"]),
            "index": rng.choice(["int64", "int32", "int16"]), "by_row": rng.random() < 0.5, "scale": rng.choice([1.0, 0.5, 11.3125])}


# ---- the 8-bit form, plain --------------------------------------------------------------------------------------------------

def _pow2(k):
    """2^k for whole k in [-126, 127], exact: the exponent's bits."""
    return ((k.to(torch.int32) + 127) << 23).view(torch.float32)


def _blocks(x):
    rows, width = x.shape
    padded = torch.nn.functional.pad(x, (0, -width % BLOCK))
    return padded.reshape(rows, -1, BLOCK)


def _round_plain(v, fmt):
    if fmt == "int8":
        return torch.round(v)
    exponent = torch.clamp((v.abs().view(torch.int32) >> 23) - 127, min=-6)
    step = _pow2(exponent - 3)
    return torch.clamp(torch.round(v / step) * step, -480.0, 480.0)


def _quantise_plain(x, fmt, keep):
    """(the numbers that the 8-bit codes stand for before scaling, the blocks' exponents), of fp32 rows."""
    b = _blocks(x)
    top, largest, smallest = (6, 127.0, 1.0) if fmt == "int8" else (8, 448.0, 2.0 ** -9)
    amax = b.abs().amax(dim=-1, keepdim=True)
    k = torch.clamp((amax.view(torch.int32) >> 23) - 127 - top, min=KMIN)
    k = torch.where(_round_plain(amax * _pow2(-k), fmt) > largest, k + 1, k)
    v = b * _pow2(-k)
    r = _round_plain(v, fmt)
    if keep:
        r = torch.where((r == 0) & (v != 0), torch.copysign(torch.full_like(v, smallest), v), r)
    return r, k


def _decode_plain(codes, scales, width):
    rows = codes.shape[0]
    values = codes.to(torch.float32).reshape(rows, -1, BLOCK) * _pow2(scales.to(torch.int32) - 127).unsqueeze(-1)
    return values.reshape(rows, -1)[:, :width]


def _checkpoint(x, fmt, keep):
    """Codes and scale bytes of a checkpoint as the framework lays them out: rows padded to whole blocks, scale 2^(byte - 127)."""
    r, k = _quantise_plain(x, fmt, keep)
    codes = r.reshape(x.shape[0], -1).to(torch.int8 if fmt == "int8" else torch.float8_e4m3fn)
    return codes.contiguous(), (k.squeeze(-1) + 127).to(torch.uint8).contiguous()


# ---- inputs -----------------------------------------------------------------------------------------------------------------

def _activations(g, rows, width, dev):
    """Rows as a layer sees them: channels of uneven strength, a few rows much larger than the rest."""
    gain = torch.exp(0.7 * torch.randn(width, generator=g, device=dev))
    x = torch.randn(rows, width, generator=g, device=dev) * gain
    return x * torch.exp(0.5 * torch.randn(rows, 1, generator=g, device=dev))


def _indices(g, case, dev, padding):
    """Codes of uneven use; with padding, one in about a hundred is -1 (a place that holds no token)."""
    rows, pq, k = case["rows"], case["pq"], case["k"]
    u = torch.rand(pq, rows, generator=g, device=dev)
    idx = torch.clamp((u * u * k).to(torch.int64), max=k - 1)
    shuffle = torch.stack([torch.randperm(k, generator=g, device=dev) for _ in range(pq)])
    idx = torch.gather(shuffle, 1, idx)
    if padding:
        idx = torch.where(torch.rand(pq, rows, generator=g, device=dev) < 0.01, torch.full_like(idx, -1), idx)
    return idx


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    state = {"case": case}
    rows = case["rows"]
    if case["op"] == "pack":
        x = _activations(g, rows, case["width"], dev)
        if case["keep"]:  # the second half has been through a ReLU
            half = case["width"] // 2
            x[:, half:] = torch.clamp(x[:, half:], min=0.0)
        state["x"] = x.to(TYPES[case["type"]])
    elif case["op"] == "wgrad":
        state["a"] = (torch.randn(rows, case["m"], generator=g, device=dev) * 1e-3).to(torch.bfloat16)
        state["codes"], state["scales"] = _checkpoint(_activations(g, rows, case["n"], dev), case["fmt"], False)
        if case["relu"]:
            state["h_codes"], state["h_scales"] = _checkpoint(torch.clamp(_activations(g, rows, case["m"], dev), min=0.0), case["fmt"], True)
    elif case["op"] == "pq":
        width = case["pq"] * case["d"]
        state["codes"], state["scales"] = _checkpoint(_activations(g, rows, width, dev), case["fmt"], False)
        state["books"] = torch.randn(case["pq"], case["k"], case["d"], generator=g, device=dev) / math.sqrt(case["d"])
        state["idx"] = _indices(g, case, dev, False)
        state["g_zq"] = torch.randn(rows, width, generator=g, device=dev) * 1e-5 if case["gzq"] else None
        state["g_vq"] = torch.rand((), generator=g, device=dev) + 0.5
    else:
        idx = _indices(g, case, dev, True).to(INTS[case["index"]])
        # by_row: the index dump's layout, one row of pq indices a token, seen as (pq, rows)
        state["idx"] = idx.t().contiguous().t() if case["by_row"] else idx
        if case["op"] == "lookup":
            state["books"] = torch.randn(case["pq"], case["k"], case["d"], generator=g, device=dev).to(TYPES[case["type"]])
        else:
            state["g"] = (torch.randn(rows, case["pq"] * case["d"], generator=g, device=dev) * 1e-2).to(TYPES[case["type"]])
    return state


# ---- one pass ---------------------------------------------------------------------------------------------------------------

def _native():
    import equss_amd
    return equss_amd.native


def _pack(state, case):
    x = state["x"]
    if own:
        native = _native()
        return native.ckpt_unpack(native.ckpt_pack(x, case["fmt"], keep_sign=case["keep"]), x.dtype)
    r, k = _quantise_plain(x.to(torch.float32), case["fmt"], case["keep"])
    return (r * _pow2(k)).reshape(x.shape[0], -1)[:, :x.shape[1]].to(x.dtype)


def _wgrad(state, case):
    if own:
        native = _native()
        kept = native.ActCheckpoint(state["codes"], state["scales"], case["n"])
        relu = native.ActCheckpoint(state["h_codes"], state["h_scales"], case["m"]) if case["relu"] else None
        return native.gemm_tn_ckpt(state["a"], kept, relu=relu, want_bias=True)
    a = state["a"].to(torch.float32)
    if case["relu"]:
        a = a * (_decode_plain(state["h_codes"], state["h_scales"], case["m"]) > 0)
    return a.t().contiguous() @ _decode_plain(state["codes"], state["scales"], case["n"]), a.sum(dim=0)


def _pq(state, case):
    beta, book = 0.25, 1.0
    if own:
        native = _native()
        kept = native.ActCheckpoint(state["codes"], state["scales"], case["pq"] * case["d"])
        return native.pq_st_backward_ckpt(kept, state["books"], state["idx"], state["g_zq"], state["g_vq"], beta, book)
    rows, pq, k, d = case["rows"], case["pq"], case["k"], case["d"]
    z = _decode_plain(state["codes"], state["scales"], pq * d).reshape(rows, pq, d)
    flat = (state["idx"] + torch.arange(pq, device=z.device).unsqueeze(1) * k).t().reshape(-1)
    emb = state["books"].reshape(pq * k, d)[flat].reshape(rows, pq, d)
    norm = z.square().sum(dim=-1, keepdim=True).sqrt().clamp_min(1e-12)
    zn = z / norm
    s = state["g_vq"] * (2.0 / (float(rows) * d * pq))
    diff = zn - emb
    dzn = diff * (beta * s)
    if case["gzq"]:
        dzn = dzn + state["g_zq"].reshape(rows, pq, d)
    dz = (dzn - zn * (zn * dzn).sum(dim=-1, keepdim=True)) / norm
    g_books = torch.zeros(pq * k, d, device=z.device).index_add_(0, flat, (diff * (-book * s)).reshape(rows * pq, d))
    return dz.reshape(rows, pq * d), g_books.reshape(pq, k, d)


def _flat(idx, k):
    """Rows of the stacked codebooks, pq * k where the index is none."""
    pq = idx.shape[0]
    idx = idx.to(torch.int64)
    at = idx + torch.arange(pq, device=idx.device).unsqueeze(1) * k
    return torch.where((idx >= 0) & (idx < k), at, torch.full_like(at, pq * k)).t().reshape(-1)


def _lookup(state, case):
    if own:
        return _native().code_lookup(state["idx"], state["books"], scale=case["scale"])
    pq, k, d = case["pq"], case["k"], case["d"]
    table = torch.cat((state["books"].reshape(pq * k, d), state["books"].new_zeros(1, d))).to(torch.float32)
    out = table[_flat(state["idx"], k)] * case["scale"]
    return out.reshape(case["rows"], pq * d).to(TYPES[case["type"]])


def _lookup_grad(state, case):
    if own:
        return _native().code_lookup_grad(state["g"], state["idx"], case["k"], scale=case["scale"])
    pq, k, d = case["pq"], case["k"], case["d"]
    g = state["g"].to(torch.float32).reshape(-1, d) * case["scale"]
    return torch.zeros(pq * k + 1, d, device=g.device).index_add_(0, _flat(state["idx"], k), g)[:-1].reshape(pq, k, d)


def run(state):
    case = state["case"]
    return {"pack": _pack, "wgrad": _wgrad, "pq": _pq, "lookup": _lookup, "lookup_grad": _lookup_grad}[case["op"]](state, case)


def work(case):
    """What each pass has to read, write and compute: inputs and outputs once, the checkpoint's own bytes where it is written or read."""
    rows, op = case["rows"], case["op"]
    kept = lambda width: rows * (width + -(-width // BLOCK))  # noqa: E731
    if op == "pack":
        return {"bytes": 2 * rows * case["width"] * BYTES[case["type"]] + 2 * kept(case["width"]), "flops": 0}
    if op == "wgrad":
        m, n = case["m"], case["n"]
        return {"bytes": 2 * rows * m + kept(n) + (rows * m if case["relu"] else 0) + 4 * m * n + 4 * m, "flops": 2 * rows * m * n}
    pq, k, d = case["pq"], case["k"], case["d"]
    cells = rows * pq * d
    if op == "pq":
        return {"bytes": kept(pq * d) + 8 * rows * pq + 4 * cells * (2 if case["gzq"] else 1) + 8 * pq * k * d, "flops": 14 * cells}
    index, value = BYTES[case["index"]] * rows * pq, BYTES[case["type"]]
    if op == "lookup":
        return {"bytes": index + value * cells + value * min(rows, k) * pq * d, "flops": cells}
    return {"bytes": index + value * cells + 4 * pq * k * d, "flops": 2 * cells}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------

def _pow2_64(k):
    return ((k.to(torch.int64) + 1023) << 52).view(torch.float64)


def _kept_exact(x, fmt, keep):
    """The kept values of fp64 rows, by the definition: candidates for k are tried from below until the largest magnitude fits."""
    rows, width = x.shape
    x = torch.cat((x, x.new_zeros(rows, -width % BLOCK)), dim=1).reshape(-1, BLOCK)

    def nearest(v):
        if fmt == "int8":
            return torch.round(v)
        _, e = torch.frexp(v)                                  # v = m 2^e, 0.5 <= m < 1: three bits behind the first
        step = _pow2_64(torch.clamp(e - 1, min=-6) - 3)
        return torch.round(v / step) * step

    peak, limit = x.abs().max(dim=1).values, 127.0 if fmt == "int8" else 448.0
    _, e = torch.frexp(peak)
    k = torch.clamp(e.to(torch.int64) - (9 if fmt == "int8" else 11), min=KMIN)
    for _ in range(4):
        k = k + (nearest(peak * _pow2_64(-k)) > limit)
    v = x * _pow2_64(-k).unsqueeze(1)
    r = nearest(v)
    if keep:
        r = r + (r == 0) * torch.sign(v) * (1.0 if fmt == "int8" else 2.0 ** -9)
    return (r * _pow2_64(k).unsqueeze(1)).reshape(rows, -1)[:, :width]


def _values_exact(codes, scales, width):
    s = _pow2_64(scales.to(torch.int64) - 127).repeat_interleave(BLOCK, dim=1)
    return (codes.to(torch.float32).to(torch.float64) * s)[:, :width]


def exact(case, seed):
    state = prepare(case, seed)
    op, rows = case["op"], case["rows"]
    if op == "pack":
        return _kept_exact(state["x"].to(torch.float64), case["fmt"], case["keep"])
    if op == "wgrad":
        a = state["a"].to(torch.float64)
        if case["relu"]:
            a = torch.where(_values_exact(state["h_codes"], state["h_scales"], case["m"]) > 0, a, torch.zeros_like(a))
        b = _values_exact(state["codes"], state["scales"], case["n"])
        return torch.mm(a.t().contiguous(), b), torch.sum(a, 0)
    pq, k, d = case["pq"], case["k"], case["d"]
    idx = state["idx"].to(torch.int64)
    if op == "pq":
        z = _values_exact(state["codes"], state["scales"], pq * d)
        s = float(state["g_vq"]) * 2.0 / (rows * d * pq)
        dz, db = torch.zeros_like(z), torch.zeros(pq, k, d, dtype=torch.float64, device=z.device)
        for p in range(pq):
            cols = slice(p * d, (p + 1) * d)
            book = state["books"][p].to(torch.float64)
            emb = book[idx[p]]
            length = torch.linalg.vector_norm(z[:, cols], dim=1, keepdim=True).clamp_min(1e-12)
            unit = z[:, cols] / length
            into = 0.25 * s * (unit - emb)
            if case["gzq"]:
                into = into + state["g_zq"][:, cols].to(torch.float64)
            dz[:, cols] = (into - unit * (unit * into).sum(1, keepdim=True)) / length
            uses = torch.bincount(idx[p], minlength=k).to(torch.float64).unsqueeze(1)
            db[p] = s * (uses * book - torch.zeros_like(book).index_add_(0, idx[p], unit))
        return dz, db
    held = (idx >= 0) & (idx < k)
    if op == "lookup":
        out = torch.zeros(rows, pq, d, dtype=torch.float64, device=idx.device)
        for p in range(pq):
            out[held[p], p] = state["books"][p].to(torch.float64)[idx[p][held[p]]] * case["scale"]
        return out.reshape(rows, pq * d)
    g = state["g"].to(torch.float64).reshape(rows, pq, d) * case["scale"]
    sums = torch.zeros(pq, k, d, dtype=torch.float64, device=idx.device)
    for p in range(pq):
        sums[p].index_add_(0, idx[p][held[p]], g[held[p], p])
    return sums
