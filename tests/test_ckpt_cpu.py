"""Refusals of the 8-bit checkpoint and codeword-lookup calls, and what they do before any launch: no GPU needed, nothing is
dereferenced on these paths."""
import ctypes

import pytest
import torch

FAKE = ctypes.c_void_p(1 << 20)      # non-null, aligned, never dereferenced
NULL, SHAPE, UNSUPPORTED, ALIGN, WORKSPACE = 1, 2, 3, 4, 5


def test_pack_and_unpack_check_their_arguments(native):
    lib = native.load_library()

    def pack(x=FAKE, type=0, ld_x=100, codes=FAKE, ld_codes=128, scales=FAKE, ld_scales=4, rows=10, width=100, fmt=0):
        got = lib.equss_ckpt_pack(x, type, ld_x, codes, ld_codes, scales, ld_scales, rows, width, fmt, 0, None)
        assert got == lib.equss_ckpt_unpack(codes, ld_codes, scales, ld_scales, x, type, ld_x, rows, width, fmt, None)
        return got

    assert pack(x=None) == pack(codes=None) == pack(scales=None) == NULL
    assert pack(rows=-1) == pack(width=0) == SHAPE
    assert pack(type=3) == pack(fmt=2) == pack(width=1 << 20, ld_x=1 << 20, ld_codes=1 << 20, ld_scales=1 << 15) == UNSUPPORTED
    assert pack(ld_x=99) == pack(ld_codes=96) == pack(ld_codes=132) == pack(ld_scales=3) == ALIGN
    assert pack(codes=ctypes.c_void_p((1 << 20) + 8)) == pack(x=ctypes.c_void_p((1 << 20) + 2)) == ALIGN
    assert b"multiple of 32" in lib.equss_last_error()
    assert pack(rows=0, x=None, codes=None, scales=None) == 0          # nothing to do, nothing launched


def test_weight_gradient_checks_its_arguments(native):
    lib = native.load_library()
    big = 1 << 34

    def grad(a=FAKE, lda=256, codes=FAKE, ld_codes=128, scales=FAKE, ld_scales=4, fmt=0, relu=None, ld_relu=0, c=FAKE, ldc=100, rows=100000,
             m=256, n=100, ws=FAKE, ws_bytes=big):
        return lib.equss_gemm_tn_ckpt(a, lda, codes, ld_codes, scales, ld_scales, fmt, relu, ld_relu, c, ldc, None, rows, m, n, ws, ws_bytes, None)

    assert grad(a=None) == grad(codes=None) == grad(scales=None) == grad(c=None) == NULL
    assert grad(rows=-1) == grad(m=0) == grad(n=0) == SHAPE
    assert grad(fmt=7) == UNSUPPORTED
    assert grad(lda=255) == grad(ld_codes=96) == grad(ld_codes=130) == grad(ld_scales=3) == grad(ldc=99) == ALIGN
    assert grad(relu=FAKE, ld_relu=255) == grad(relu=FAKE, ld_relu=224) == grad(relu=ctypes.c_void_p((1 << 20) + 4), ld_relu=256) == ALIGN
    need = lib.equss_gemm_tn_ckpt_workspace_bytes(100000, 256, 100)
    assert need > 0
    assert grad(ws=None) == grad(ws_bytes=need - 1) == grad(ws=ctypes.c_void_p((1 << 20) + 8)) == WORKSPACE
    assert lib.equss_gemm_tn_ckpt_workspace_bytes(64, 256, 100) == 0     # one row range: straight into C
    assert lib.equss_gemm_tn_ckpt_workspace_bytes(0, 256, 100) == lib.equss_gemm_tn_ckpt_workspace_bytes(10, 0, 100) == 0


def test_quantiser_backward_checks_its_arguments(native):
    lib = native.load_library()
    f = ctypes.c_float
    big = 1 << 34

    def back(codes=FAKE, ld_codes=1024, scales=FAKE, ld_scales=32, fmt=0, books=FAKE, idx=FAKE, g_zq=None, ld_g=0, g_vq=FAKE, g_z=FAKE, ld_gz=1024,
             g_books=FAKE, rows=10000, num_pq=8, k=256, d=128, ws=FAKE, ws_bytes=big):
        return lib.equss_pq_st_backward_ckpt(codes, ld_codes, scales, ld_scales, fmt, books, idx, g_zq, ld_g, g_vq, f(0.25), f(1.0), g_z, ld_gz,
                                             g_books, rows, num_pq, k, d, ws, ws_bytes, None)

    assert back(codes=None) == back(scales=None) == back(books=None) == back(idx=None) == back(g_vq=None) == NULL
    assert back(rows=0) == back(num_pq=0) == back(k=0) == SHAPE
    assert back(d=48) == back(fmt=2) == back(rows=(1 << 31) - 200) == UNSUPPORTED
    assert back(ld_codes=992) == back(ld_scales=31) == back(ld_gz=1020) == back(g_zq=FAKE, ld_g=1022) == ALIGN
    assert back(g_books=ctypes.c_void_p((1 << 20) + 4)) == back(books=ctypes.c_void_p((1 << 20) + 4)) == ALIGN
    need = lib.equss_code_sums_sorted_workspace_bytes(10000, 8, 256, 128)
    assert need > 0 and back(ws=None) == back(ws_bytes=need - 1) == back(ws=ctypes.c_void_p((1 << 20) + 64)) == WORKSPACE
    assert back(g_z=None, g_books=None) == 0                             # nothing wanted, nothing launched


def test_lookup_and_its_gradient_check_their_arguments(native):
    lib = native.load_library()
    f = ctypes.c_float

    def look(idx=FAKE, it=0, books=FAKE, type=0, out=FAKE, ld_out=64, rows=10, num_pq=4, k=20, d=16):
        return lib.equss_code_lookup(idx, it, rows, 1, books, type, f(1.0), out, ld_out, rows, num_pq, k, d, None)

    assert look(idx=None) == look(books=None) == look(out=None) == NULL
    assert look(rows=-1) == look(num_pq=0) == look(k=0) == look(d=0) == SHAPE
    assert look(it=3) == look(type=3) == look(k=1 << 31) == look(rows=(1 << 31) - 1) == look(num_pq=70000, ld_out=70000 * 16) == look(num_pq=1, d=1 << 24, ld_out=1 << 24) == UNSUPPORTED
    assert look(ld_out=63) == look(books=ctypes.c_void_p((1 << 20) + 4)) == look(out=ctypes.c_void_p((1 << 20) + 2)) == ALIGN
    assert look(rows=0, idx=None, books=None, out=None) == 0

    def grad(g=FAKE, type=0, ld_g=64, idx=FAKE, it=0, out=FAKE, rows=5000, num_pq=4, k=20, d=16, ws=FAKE, ws_bytes=1 << 34):
        return lib.equss_code_lookup_grad(g, type, ld_g, idx, it, rows, 1, f(1.0), out, rows, num_pq, k, d, ws, ws_bytes, None)

    assert grad(g=None) == grad(idx=None) == grad(out=None) == NULL
    assert grad(rows=-1) == grad(d=0) == SHAPE
    assert grad(it=-1) == grad(type=5) == grad(k=1 << 31) == grad(rows=(1 << 31) - 1) == UNSUPPORTED
    assert grad(ld_g=63) == grad(out=ctypes.c_void_p((1 << 20) + 8)) == grad(g=ctypes.c_void_p((1 << 20) + 1)) == ALIGN
    assert grad(ws=None) == grad(ws_bytes=100) == WORKSPACE


def test_python_calls_refuse_before_they_reach_the_library(native):
    x = torch.zeros(4, 40)
    for call in (lambda: native.ckpt_pack(x), lambda: native.code_lookup(torch.zeros(1, 4, dtype=torch.long), torch.zeros(1, 3, 8)),
                 lambda: native.code_lookup_grad(x, torch.zeros(1, 4, dtype=torch.long), 3)):
        with pytest.raises(native.EqussError):        # host tensors: there is no CPU path
            call()
    codes, scales = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.uint8)
    kept = native.ActCheckpoint(codes, scales, 40)
    assert (kept.rows, kept.width, kept.fmt) == (4, 40, "int8")
    assert native.ActCheckpoint(codes.view(torch.float8_e4m3fn), scales, 64).fmt == "e4m3"
    part = kept.columns(32, 40)
    assert part.codes.shape == (4, 32) and part.scales.shape == (4, 1) and part.width == 8
    for bad in (lambda: native.ActCheckpoint(codes, scales, 65), lambda: native.ActCheckpoint(codes, scales, 32), lambda: native.ActCheckpoint(codes.float(), scales, 40),
                lambda: native.ActCheckpoint(codes, scales[:, :1], 40), lambda: native.ActCheckpoint(codes, scales.long(), 40), lambda: kept.columns(8, 40),
                lambda: kept.columns(0, 33), lambda: kept.columns(32, 32), lambda: kept.columns(0, 41), lambda: native.ActCheckpoint(codes, scales, 0)):
        with pytest.raises(ValueError):
            bad()
