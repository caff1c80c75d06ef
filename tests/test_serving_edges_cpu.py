"""The serving operators without a GPU: more that the C entry points refuse before anything is
launched, and what their sources must not hold."""
import os

import pytest

from megakernel_b200 import _lib, build
from test_serving_cpu import INVALID, append


@pytest.mark.parametrize("kw", [dict(k_stride=[4096, 0, 128]), dict(v_stride=[4096, 0, 128]),
                                dict(k_stride=[0, 2048, 128]), dict(v_stride=[4096, 2048, 0])])
def test_append_refuses_rows_at_one_place(kw):
    """Strides of 0 between KV heads, pages or slots: several rows would be written to the same memory."""
    assert _lib.load().mkb_paged_append(append(**kw), None) == INVALID


@pytest.mark.parametrize("source", ["mkb_append.cu", "mkb_attn_tc.cu", "mkb_attn_decode.cu", "mkb_serving.cuh"])
def test_kernels_that_start_early_use_coherent_loads(source):
    """These kernels are brought in while the one before them in the stream still runs. A load of
    data that has to be read-only for the kernel's whole life (ld.global.nc) would be of memory
    that the one before may be writing, as the append writes a decode step's q."""
    with open(os.path.join(build.CSRC, source)) as f:
        text = f.read()
    assert "__ldg(" not in text and "__restrict__" not in text and ".nc" not in text
