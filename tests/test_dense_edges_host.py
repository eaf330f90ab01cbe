"""The dense side without a GPU, further: refusals before any launch."""

import pytest

from test_dense_host import FAKE, ST, call, lib, strides  # noqa: F401


@pytest.mark.parametrize("dims,grid", [((128, 0, 0), (2 ** 26, 1, 1)), ((0, 128, 0), (1, 2 ** 26, 1)), ((44, 42, 42), (1, 1, 2 ** 27)),
                                       ((0, 0, 128), (2 ** 10, 1, 2 ** 25))])
def test_rope_tables_beyond_32_bits(lib, dims, grid):  # noqa: F811
    """The kernels index an axis's table of cosines with 32 bits."""
    rope = [FAKE, *dims, *grid, 0]
    args = [FAKE, strides(*ST), 2, FAKE, FAKE, None, None, 0, None, None, 2, 0, 1, 64, 128, 1e-6, *rope, None]
    rc, msg = call(lib, "bsa_norm_rope", "psipppsippiiiiifpiiiiiiip", args)
    assert rc == 1 and "table" in msg
    args = [FAKE, strides(*ST), FAKE, strides(*ST), 2, FAKE, FAKE, None, None, None, None, None, 0, None, None, None, 2, 0, 1, 64, 128,
            1e-6, *rope, None, None]
    rc, msg = call(lib, "bsa_norm_rope_backward", "pspsippppspsipppiiiiifpiiiiiiipp", args)
    assert rc == 1 and "table" in msg


def test_rope_places_beyond_32_bits(lib):  # noqa: F811
    """A grid may hold more than 2^31 places; the tokens' own stay within 32 bits."""
    rope = [FAKE, 44, 42, 42, 2 ** 11, 2 ** 10, 2 ** 11, 2 ** 31 - 32]
    args = [FAKE, strides(*ST), 2, FAKE, FAKE, None, None, 0, None, None, 2, 0, 1, 64, 128, 1e-6, *rope, None]
    rc, msg = call(lib, "bsa_norm_rope", "psipppsippiiiiifpiiiiiiip", args)
    assert rc == 1 and "32 bits" in msg


def test_tokens_at_the_32_bit_border(lib):  # noqa: F811
    """The last tile's rows behind the last token are counted in 32 bits too."""
    args = [FAKE, strides(8, 8, 8), 1, FAKE, FAKE, None, None, 0, None, None, 2, 0, 1, 2 ** 31 - 3, 8, 1e-6, None, 0, 0, 0, 0, 0, 0, 0,
            None]
    rc, msg = call(lib, "bsa_norm_rope", "psipppsippiiiiifpiiiiiiip", args)
    assert rc == 1 and "too many tokens" in msg
