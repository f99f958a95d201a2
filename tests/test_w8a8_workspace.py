"""CPU: where the 8-bit linear puts its codes in a caller's workspace (every call here is refused before
any launch; addresses are never read)."""

from __future__ import annotations

import pytest

P, FAR, BF16 = 4096, 1 << 30, 2


@pytest.fixture(scope="module")
def lib():
    from convrot_mlx_amd import _native

    return _native.load()


@pytest.mark.parametrize("nbytes", [22 * 1024, 32 * 1024, 36 * 1024, 37 * 1024])
def test_codes_stay_off_the_control_block(lib, nbytes):
    """40 rows of 64 features need 5280 bytes: at most a quarter of these workspaces, but what they leave is
    less than the 32 KiB of the control block, whose counters stay zero between launches."""
    assert lib.convrot_w8a8_scratch_bytes(40, 64) == 5280 <= nbytes // 4
    rc = lib.convrot_w8a8_linear(P, BF16, 64, P, 64, P, None, 40, 8, 64, None, None, 0, 1, None, 0, P, nbytes, FAR, None)
    assert rc == 1 and "scratch buffer of 5280 bytes" in lib.convrot_last_error().decode()


def test_workspace_bytes_of_a_product(lib):
    """32 KiB and the partial sums where workgroups share K, nothing where they do not, never more than the
    workspace of the other linears."""
    most = lib.convrot_w4a4_workspace_bytes()
    for m, n, k in ((1, 512, 8192), (4, 1024, 12288), (16, 64, 65536), (24, 3072, 12288), (40, 96, 12288), (128, 4096, 16384)):
        need = lib.convrot_w8a8_workspace_bytes(m, n, k)
        assert 32768 + 2 * 4096 <= need <= most and need % 4096 == 0
    for m, n, k in ((1, 18432, 3072), (77, 9216, 3072), (4608, 12288, 3072), (3, 64, 128), (0, 64, 128), (4, 64, 0),
                    (4, 64, 65552)):
        assert lib.convrot_w8a8_workspace_bytes(m, n, k) == 0


def test_workspace_bytes_of_what_no_launch_takes(lib):
    assert lib.convrot_w8a8_workspace_bytes(0x7ffffe00, 0x7ffffe00, 64) == 0
    try:
        assert lib.convrot_set_tuning(b"w8a8_tile", b"64x64") == 0
        assert lib.convrot_w8a8_workspace_bytes(1 << 30, 1 << 20, 64) == 0
    finally:
        lib.convrot_set_tuning(b"w8a8_tile", None)
