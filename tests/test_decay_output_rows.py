"""Outputs whose rows share elements are refused before any device is touched."""
import ctypes

import pytest
import torch

# (token stride, head stride) of 4 tokens of 2 heads of 64, and whether their rows lie apart
LAYOUTS = [((128, 64), True), ((64, 256), True), ((192, 96), True), ((200, 100), True), ((64, 264), True),
           ((0, 64), False), ((128, 0), False), ((64, 64), False), ((126, 64), False), ((128, 60), False),
           ((64, 250), False), ((60, 512), False)]


@pytest.mark.parametrize("strides,apart", LAYOUTS)
def test_entry_points_refuse_overlapping_outputs(strides, apart):
    if apart and torch.cuda.is_available():
        pytest.skip("the call would run")
    from catfuse_b200 import _lib
    lib = _lib.load()
    good, st = (128, 64), strides
    # addresses are never followed: the last refusal is that there is no device
    rcs = [lib.cf_decay_attention(16, 16, 16, 64, 1, 16, None, None, None, 0, None, 1, 4, 4, 2, 2, 64, 64,
                                  *good, *good, *good, *st, 1.0, None, 0, None),
           lib.cf_decay_attention_step(16, 16, 16, 64, 1, 16, 16, 16, None, 4, 4, 2, 2, 64, 64,
                                       *good, *good, *good, *st, 1.0, None)]
    for outs in ((st, good), (good, st)):
        rcs.append(lib.cf_qk_norm_rope(16, 16, 16, 16, 1, 4, 2, 2, 64, *good, *good, *outs[0], *outs[1], 16, 32, 4,
                                       16, 64, (ctypes.c_int32 * 1)(32), 1, 0, 0, None, None, 1, 1e-6, None))
    # without tokens there are no rows
    if not torch.cuda.is_available():
        rc = lib.cf_decay_attention(None, None, None, None, 1, 16, None, None, None, 0, None, 1, 0, 0, 2, 2, 64, 64,
                                    *good, *good, *good, 0, 0, 1.0, None, 0, None)
        assert rc == _lib.CF_ERR_NO_DEVICE
    for rc in rcs:
        assert rc == (_lib.CF_ERR_NO_DEVICE if apart else _lib.CF_ERR_INVALID_ARG), _lib.last_error()


def test_entry_points_refuse_outputs_in_place_of_q_or_k():
    """The CTAs of a head's 32 columns each share its q and k, so none may write there (rows
    on 16 bytes of a prompt have one CTA a head, which reads them first)."""
    from catfuse_b200 import _lib
    lib = _lib.load()
    st = (128, 64) * 4
    for q, k in ((64, 32), (32, 64)):
        assert lib.cf_decay_attention_step(q, k, 16, 64, 1, 16, 16, 16, None, 4, 4, 2, 2, 64, 64,
                                           *st, 1.0, None) == _lib.CF_ERR_INVALID_ARG
        assert lib.cf_decay_attention(q + 2, k + 2, 16, 66, 1, 16, None, None, None, 0, None, 1, 4, 4, 2, 2, 64, 64,
                                      *st, 1.0, None, 0, None) == _lib.CF_ERR_INVALID_ARG
