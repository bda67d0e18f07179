"""The calls that make an autograd node's forward and backward record nothing, and refuse tensors that want it recorded
(the launch patched out; no GPU needed)."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import nanopysche_amd as fm
from tests.test_host_act8_balance import act
from tests.test_host_decode_int8 import launched  # noqa: F401

BF = torch.bfloat16


def calls(x, w):
    """Each call with x (and w) in every place that a gradient could come from."""
    plain, ones, r = torch.zeros(2, 32, dtype=BF), torch.ones(32), torch.ones(2)
    wide = torch.cat((x, x), 1)
    return {"swiglu_compress": [lambda: fm.swiglu_compress(wide), lambda: fm.swiglu_compress(x, plain), lambda: fm.swiglu_compress(plain, x)],
            "swiglu_backward_8bit": [lambda: fm.swiglu_backward_8bit(x, act(2, 32), act(2, 32)),
                                     lambda: fm.swiglu_backward_8bit(x, act(2, 32), act(2, 32), packed=True)],
            "rmsnorm_compress": [lambda: fm.rmsnorm_compress(x, ones), lambda: fm.rmsnorm_compress(plain, w)],
            "rmsnorm_backward_8bit": [lambda: fm.rmsnorm_backward_8bit(x, act(2, 32), ones, r, need_dw=False),
                                      lambda: fm.rmsnorm_backward_8bit(plain, act(2, 32), w, r, need_dw=False)]}


def test_gradients_are_refused(launched):  # noqa: F811
    x, w = torch.zeros(2, 32, dtype=BF, requires_grad=True), torch.ones(32, requires_grad=True)
    for name, group in calls(x, w).items():
        for call in group:
            with pytest.raises(RuntimeError, match=f"{name} records no gradient"):
                call()
    assert launched == []


def test_tangents_are_refused(launched):  # noqa: F811
    with fwAD.dual_level():
        x = fwAD.make_dual(torch.zeros(2, 32, dtype=BF), torch.ones(2, 32, dtype=BF))
        w = fwAD.make_dual(torch.ones(32), torch.ones(32))
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for name, group in calls(x, w).items():
                    for call in group:
                        with pytest.raises(RuntimeError, match=f"{name} records no tangent"):
                            call()
    assert launched == []


def test_without_recording_they_run(launched):  # noqa: F811
    x, w = torch.zeros(2, 32, dtype=BF, requires_grad=True), torch.ones(32, requires_grad=True)
    with torch.no_grad():
        made = [call() for group in calls(x, w).values() for call in group]
    made += [call() for group in calls(x.detach(), w.detach()).values() for call in group]
    assert len(launched) == len(made) == 18
    for name in ("fm_act8_swiglu", "fm_act8_swiglu_backward", "fm_act8_rmsnorm", "fm_act8_rmsnorm_backward"):
        assert name in launched


def test_what_is_kept_carries_none(launched):  # noqa: F811
    """compress_activation keeps a leaf of a step that is being recorded."""
    x = torch.zeros(2, 32, dtype=BF, requires_grad=True)
    t = fm.compress_activation(x)
    assert not t.data.requires_grad and not t.restore().requires_grad
