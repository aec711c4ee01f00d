"""What the checkpoint and lookup calls decide on the host, at the ends of their sizes: no GPU needed."""
import ctypes

import torch


def test_partial_sums_of_wide_codewords_go_by_all_their_columns(native):
    """8192 rows of 4096 columns fill the chip with tiles of 32: 256 tiles with two partial sums of 4096 floats each, beside 8
    bytes a row and the sort's tables."""
    lib = native.load_library()
    got = lib.equss_code_sums_sorted_workspace_bytes(8192, 1, 256, 4096)
    assert 256 * 2 * 4096 * 4 <= got <= 256 * 2 * 4096 * 4 + 8192 * 8 + 64 * 2048 * 4 + 4096, got


def test_sizes_past_a_launch_are_refused_before_it(native):
    """A dimension of a launch has fewer than 2^32 threads."""
    lib = native.load_library()
    p = ctypes.c_void_p(1 << 20)         # non-null, aligned, never dereferenced
    UNSUPPORTED, wide = 3, 1 << 19
    assert lib.equss_ckpt_pack(p, 0, wide, p, wide, p, wide // 32, 1 << 24, wide, 0, 0, None) == UNSUPPORTED
    assert lib.equss_ckpt_unpack(p, wide, p, wide // 32, p, 0, wide, 1 << 24, wide, 0, None) == UNSUPPORTED
    assert lib.equss_code_lookup(p, 0, 1 << 24, 1, p, 0, ctypes.c_float(1.0), p, 1 << 14, 1 << 24, 1, 4, 1 << 14, None) == UNSUPPORTED

    def grad(m, n):
        return lib.equss_gemm_tn_ckpt(p, m, p, (n + 31) // 32 * 32, p, (n + 31) // 32, 0, None, 0, p, n, None, 1, m, n, p, 1 << 62, None)

    assert grad(1 << 20, 1 << 20) == grad(8, (1 << 31) - 1) == grad((1 << 31) - 1, 8) == grad((1 << 30) + 1, 8) == UNSUPPORTED
    assert lib.equss_gemm_tn_ckpt_workspace_bytes(1 << 20, (1 << 31) - 1, 8) == lib.equss_gemm_tn_ckpt_workspace_bytes(1 << 20, 8, (1 << 31) - 1) == 0


def test_modules_saved_whole_before_they_had_the_setting(pkg, tmp_path):
    """A pickled module brings its own attributes and nothing else: the setting's default comes from the class."""
    model = pkg.build_model(pkg.configs.pqgo_config())
    block = model.model.vq_blocks[0]
    for module in (model.model, block, *block.quantizers):
        for name in ("activation_checkpoint", "_activation_checkpoint"):
            module.__dict__.pop(name, None)
    torch.save(model, tmp_path / "model.pt")
    back = torch.load(tmp_path / "model.pt", weights_only=False)            # (this test's own file)
    block = back.model.vq_blocks[0]
    assert back.model.activation_checkpoint == block.activation_checkpoint == block.quantizers[0].activation_checkpoint == "none"
    back.model.activation_checkpoint = "e4m3"
    assert back.model.activation_checkpoint == block.activation_checkpoint == "e4m3"
