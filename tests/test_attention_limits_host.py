"""The diagnostic limit of the attention's waits, without a GPU: what it takes and refuses."""
import pytest

from dcnv2_b200 import capi
from dcnv2_b200.capi import DCNv2Error, Status, lib


def test_wait_limit_range():
    for bad in (-2, 2000001, -2 ** 31, 2 ** 31 - 1):
        assert lib.dcnv2_diag_set_attention_wait_limit(bad) == Status.ERR_INVALID_ARG
    for good in (0, 1000, 2000000, -1):
        assert lib.dcnv2_diag_set_attention_wait_limit(good) == Status.OK
    with pytest.raises(DCNv2Error):
        capi.set_attention_wait_limit(-7)
    capi.set_attention_wait_limit()
