"""CPU: limits of the label operators, refused before anything is launched."""
import ctypes as C
import os
import re
import shutil
import subprocess

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


CALLS = [lambda z, w: A.linear_fp8(z, w), lambda z, w: A.linear_fp8(w, z), lambda z, w: A.linear_fp8(w, w, z[:, 0]), lambda z, w: A.distill_top_logits(z, w, w.long()),
         lambda z, w: A.distill_top_logits(w, z, w.long()), lambda z, w: A.distill_top_logits_grad(z, w, w.long(), w[:, 0]),
         lambda z, w: A.distill_top_logits_grad(w, w, w.long(), z[:, 0])]


@pytest.mark.parametrize("call", CALLS)
def test_forward_mode_tangents_are_refused(call, monkeypatch):
    monkeypatch.setattr(_lib, "require_cuda", lambda *a: None)                  # the checks alone, on the CPU
    z, w = torch.randn(3, 5), torch.randn(3, 5)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(torch.autograd.forward_ad.make_dual(z, torch.ones_like(z)), w)


@pytest.mark.parametrize("call", [CALLS[0], CALLS[3], CALLS[5], lambda z, w: A.sample_logits(z, w[:, 0]), lambda z, w: A.quantize_fp8(z).data])
def test_recorders_are_refused(call):
    """what they record is the allocation of the results: the replayed program would return memory that nothing has written"""
    from torch.fx.experimental.proxy_tensor import make_fx
    z, w = torch.randn(3, 5), torch.randn(3, 5)
    with pytest.raises(RuntimeError, match="recorded"):
        torch.jit.trace(call, (z, w), check_trace=False)
    with pytest.raises(RuntimeError, match="recorded"):
        make_fx(call)(z, w)
    with pytest.raises(RuntimeError, match="GPU"):
        call(z, w)


CSRC = os.path.join(os.path.dirname(os.path.abspath(A.__file__)), "csrc")


@pytest.mark.skipif(shutil.which("hipcc") is None, reason="needs the compiler")
def test_product_waits_for_its_copies_before_every_barrier(tmp_path):
    """A wave's copies from memory into LDS are read by the others behind the next barrier, so each wave has to wait for its own in front of
    it, in every instance and not where the compiler happens to.  (The one barrier in an asm block of its own, which orders reads of
    LDS alone, waits for nothing on purpose.)"""
    flags = re.search(r"^CXXFLAGS := (.*)$", open(os.path.join(CSRC, "Makefile")).read(), re.M).group(1)
    flags = [f for f in flags.replace("$(ARCH)", "gfx950").replace("$(NO_PACKED)", "-Xclang -target-feature -Xclang -packed-fp32-ops").split() if "$" not in f]
    out = str(tmp_path / "label_fp8.s")
    subprocess.run(["hipcc", *flags, "--offload-device-only", "-S", os.path.join(CSRC, "label_fp8.hip"), "-o", out], check=True, stderr=subprocess.DEVNULL)
    kernels = 0
    for name, body in re.findall(r"^(_Z\S*gemm_fp8_kernel\S*):[^\n]*\n(.*?)^\.Lfunc_end", open(out).read(), re.M | re.S):
        lines = [x.strip() for x in body.split("\n")]
        barriers = [i for i, x in enumerate(lines) if x.startswith("s_barrier")]
        assert any("global_load_lds" in x for x in lines) and len(barriers) >= 2, name
        bare = 0
        for i in barriers:
            back = i - 1
            while not re.match(r"s_waitcnt.*vmcnt\(0\)|\S+:|s_c?branch|;;#ASMEND", lines[back]):
                back -= 1
            bare += lines[back].startswith(";;#ASMEND")
            assert "vmcnt(0)" in lines[back] or lines[back].startswith(";;#ASMEND"), (name, lines[back:i + 1])
        assert bare <= 1, name
        kernels += 1
    assert kernels == 26                                        # 2 or 3 tiles x 3 result types x 4 operand types, the widened and raw forms without the largest
