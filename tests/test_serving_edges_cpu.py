"""More that the C entry points of the serving operators refuse before anything is launched."""
import pytest

from megakernel_b200 import _lib
from test_serving_cpu import INVALID, append


@pytest.mark.parametrize("kw", [dict(k_stride=[4096, 0, 128]), dict(v_stride=[4096, 0, 128]),
                                dict(k_stride=[0, 2048, 128]), dict(v_stride=[4096, 2048, 0])])
def test_append_refuses_rows_at_one_place(kw):
    """Strides of 0 between KV heads, pages or slots: several rows would be written to the same memory."""
    assert _lib.load().mkb_paged_append(append(**kw), None) == INVALID
