"""CPU: limits of the label operators, refused before anything is launched."""
import ctypes as C

import pytest
import torch

import object_nerf_amd as A
from object_nerf_amd import _lib


def _sample(**kw):
    a = _lib.SampleArgs()
    for k, v in {**dict(n=2, v=8, type=1, logits=64, logits_stride=8, u=64, u_stride=1, temperature=1.0, top_p=1.0, labels=64), **kw}.items():
        setattr(a, k, v)
    return _lib.lib().objnerf_sample_logits(C.byref(a), None)


def test_sample_refuses_rows_that_its_sums_cannot_hold():
    l = _lib.lib()
    for v in ((1 << 19) + 1, 1 << 20, (1 << 31) - 1):
        assert _sample(v=v, logits_stride=v) < 0 and b"2^19" in l.objnerf_last_error()
        assert l.objnerf_sample_logits_workspace_bytes(1, v, 1) == 0
    assert _sample(n=0, v=1 << 19) == 0
