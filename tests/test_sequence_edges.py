"""The sequence operators without a GPU: the ends of what their C entry points and tensor functions take."""
import ctypes

import pytest

from test_sequence import FAKE, attn, lib  # noqa: F401


@pytest.mark.parametrize("softcap", [1e-45, 1e-39])
def test_a_cap_whose_reciprocal_is_no_number_is_refused(lib, softcap):
    a = attn(softcap=softcap)
    assert lib.bigc_seq_attn_fwd(None, ctypes.byref(a), FAKE, 1 << 40) == -1
    assert lib.bigc_seq_attn_bwd(None, ctypes.byref(a), FAKE, 1 << 40) == -1
