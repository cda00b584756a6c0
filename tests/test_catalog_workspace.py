"""Scratch memory that the catalog's entry points ask for: a matter of arithmetic on the host, no GPU."""
import pytest

from graphsage_amd import _lib


@pytest.mark.parametrize('items', [1000, 100_000, 8_388_000, 9_000_000, 50_000_000])
@pytest.mark.parametrize('users', [1, 5, 128, 129, 255, 256])
@pytest.mark.parametrize('top', [1, 20, 64])
def test_scratch_grows_with_the_users_there_are(users, items, top):
    """A row of group maxima a user (of 32 items a group, or of 4), what 1024 blocks leave, the tables where they are laid out."""
    lib = _lib.load()
    for dtype, pieces in ((0, 3), (1, 1), (2, 2)):
        for dim, width in ((32, 32), (64, 64), (200, 256)):
            got = lib.gs_catalog_workspace(users, items, dim, dtype, top)
            maxima = 4 * users * (items // 4 + 64)
            laid_out = 2 * pieces * width * (users + items + 64)
            rest = 16 * 1024 * (users + 256) + 4 * (items + 64) + 8 * items // 32 + 4096
            assert 0 < got <= maxima + laid_out + rest
            if users == 1 and dim <= 64:                      # one user: nothing is laid out
                assert got <= maxima + 16 * 1024 + 8 * items // 32 + 4096


def test_one_user_of_a_large_catalog():
    lib = _lib.load()
    assert lib.gs_catalog_workspace(1, 9_000_000, 32, 1, 10) < 12 << 20
    assert lib.gs_catalog_workspace(1, 50_000_000, 32, 1, 10) < 60 << 20


def test_gradients_of_more_rows_than_a_launch_holds_are_refused():
    """Before anything is launched or read: the addresses are those of tables that are not there."""
    lib = _lib.load()
    at = 1 << 20
    rc = lib.gs_catalog_bwd(at, 1 << 30, at, 1 << 30, 1, 1, None, 1.0, None, at, None, None, None, at, None, None, at, 1 << 62, None)
    assert rc == -3 and b'together' in lib.gs_last_error()
