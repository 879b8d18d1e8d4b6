"""The diagnostic limit of the attention's waits, without a GPU: what it takes and refuses."""
import pytest
import torch

from dcnv2_b200 import (capi, dcnv2_cross_attention_error, dcnv2_cross_attention_workspace_size)
from dcnv2_b200.capi import DCNv2Error, Status, lib


def test_wait_limit_range():
    for bad in (-2, 2000001, -2 ** 31, 2 ** 31 - 1):
        assert lib.dcnv2_diag_set_attention_wait_limit(bad) == Status.ERR_INVALID_ARG
    for good in (0, 1000, 2000000, -1):
        assert lib.dcnv2_diag_set_attention_wait_limit(good) == Status.OK
    with pytest.raises(DCNv2Error):
        capi.set_attention_wait_limit(-7)
    capi.set_attention_wait_limit()


def test_workspace_helpers_refuse_what_the_call_refuses():
    q, k = torch.zeros(1, 40, 4, 64).half(), torch.zeros(1, 9, 2, 64).half()
    for call in (lambda: dcnv2_cross_attention_workspace_size(q, k, k),   # not on a GPU
                 lambda: dcnv2_cross_attention_error(q, k, k, None)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        dcnv2_cross_attention_workspace_size(q.float(), k.float(), k.float())
