"""Setting an attention half's weights on a B200: what is refused."""

import numpy as np
import pytest

import tritify_b200 as tb
from tritify_b200 import _native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [tb.WLEVELS + 1, -tb.WLEVELS - 1, 2 ** 31 - 1, -2 ** 31])
def test_norm_codes_beyond_their_range(ctx, bad):
    """As a layer's norm: codes outside +-WLEVELS are refused; those at its ends are taken."""
    a = tb.AttentionHalf(ctx, 64, 2, 1, 16)
    codes = np.ones(64, np.int32)
    codes[:2] = tb.WLEVELS, -tb.WLEVELS
    a.set_norm(codes, tb.Scale(1, 0), tb.Scale(0, 0))
    codes[63] = bad
    with pytest.raises(tb.KtmoeError) as e:
        a.set_norm(codes, tb.Scale(1, 0), tb.Scale(0, 0))
    assert e.value.status == _native.ERR_RANGE
