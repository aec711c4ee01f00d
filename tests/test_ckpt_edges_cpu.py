"""What the checkpoint and lookup calls decide on the host, at the ends of their sizes: no GPU needed."""


def test_partial_sums_of_wide_codewords_go_by_all_their_columns(native):
    """8192 rows of 4096 columns fill the chip with tiles of 32: 256 tiles with two partial sums of 4096 floats each, beside 8
    bytes a row and the sort's tables."""
    lib = native.load_library()
    got = lib.equss_code_sums_sorted_workspace_bytes(8192, 1, 256, 4096)
    assert 256 * 2 * 4096 * 4 <= got <= 256 * 2 * 4096 * 4 + 8192 * 8 + 64 * 2048 * 4 + 4096, got
