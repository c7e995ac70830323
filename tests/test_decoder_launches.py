"""A launch that does not happen is the call's error, whichever kernel it was of. Without a device no launch does: these
checks run only there."""
import ctypes as C

import pytest
import torch

from tests.test_decoder_ops import norm, norm_bwd, paged
from torchvulkan_amd import _abi

lib = _abi.load()


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="the calls' addresses are none")
@pytest.mark.parametrize("fn,desc", [
    ("tvk_rms_norm_fwd", norm()), ("tvk_rms_norm_fwd", norm(cols=40000, x_stride=40000, out_stride=40000)),
    ("tvk_rms_norm_bwd", norm_bwd(rows=3)), ("tvk_rms_norm_bwd", norm_bwd(dweight=None)),
    ("tvk_paged_append", paged(_abi.PagedAppendDesc, {})), ("tvk_paged_append", paged(_abi.PagedAppendDesc, {"cache_head_dim": 33})),
    ("tvk_paged_attention", paged(_abi.PagedAttentionDesc, {})),                                   # a wave or a workgroup each
    ("tvk_paged_attention", paged(_abi.PagedAttentionDesc, {"cache_table_width": 10000})),          # cut
    ("tvk_paged_attention", paged(_abi.PagedAttentionDesc, {"cache_head_dim": 40})),                # the general kernel
])
def test_a_launch_that_fails_is_reported(fn, desc):
    assert getattr(lib, fn)(C.byref(desc)) == _abi.TVK_ERR_DEVICE
    assert fn.encode() in lib.tvk_last_error()
