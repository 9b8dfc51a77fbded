"""What the entry points of 8-bit rows refuse, before anything is launched (no GPU)."""
import ctypes

import numpy as np
import pytest

from nitrorag_amd import _native as N
import row8_forms as forms

P = 4096  # a pointer that is never read: every call below is refused first
INVALID, UNSUPPORTED = N.INVALID_ARGUMENT, N.UNSUPPORTED


def refused(name, *args):
    with pytest.raises(N.NitroError) as e:
        N.call(name, *args)
    return e.value.status


@pytest.mark.parametrize("change,status", [
    ({0: None}, INVALID), ({2: None}, INVALID), ({5: None}, INVALID), ({6: None}, INVALID),
    ({3: 0.0}, INVALID), ({3: -1e-5}, INVALID), ({3: float("nan")}, INVALID), ({3: float("inf")}, INVALID),
    ({7: 0}, INVALID), ({7: -1}, INVALID), ({8: 0}, INVALID), ({8: -4}, INVALID), ({8: (1 << 30) + 1}, UNSUPPORTED)])
def test_rms_norm_row8_refuses(change, status):
    args = [P, None, P, 1e-5, None, P, P, 2, 64, None]
    for i, v in change.items():
        args[i] = v
    assert refused("nitro_rms_norm_row8", *args) == status


@pytest.mark.parametrize("name", ["nitro_row8_quantize", "nitro_row8_read"])
@pytest.mark.parametrize("change,status", [({0: None}, INVALID), ({1: None}, INVALID), ({2: None}, INVALID), ({3: 0}, INVALID),
                                           ({4: 0}, INVALID), ({4: (1 << 30) + 1}, UNSUPPORTED)])
def test_quantize_and_read_refuse(name, change, status):
    args = [P, P, P, 3, 32, None]
    for i, v in change.items():
        args[i] = v
    assert refused(name, *args) == status


@pytest.mark.parametrize("change,status", [
    ({0: None}, INVALID), ({2: 0}, INVALID), ({2: -32}, INVALID), ({2: 48}, INVALID), ({3: 0}, INVALID), ({0: P + 2}, INVALID),
    ({1: P + 1}, INVALID), ({2: (1 << 30) + 32}, UNSUPPORTED), ({3: (1 << 30) + 1}, UNSUPPORTED)])
def test_q8_weights_refuses(change, status):
    out = ctypes.c_void_p(7)
    args = [P, None, 64, 8, ctypes.byref(out)]
    for i, v in change.items():
        args[i] = v
    assert refused("nitro_q8_weights_create", *args) == status
    assert not out.value
    assert refused("nitro_q8_weights_create", P, None, 64, 8, None) == INVALID


def test_destroying_no_weights_is_fine():
    N.call("nitro_q8_weights_destroy", None)


def test_row8_matmul_refuses_null_weights():
    assert refused("nitro_row8_matmul", None, P, P, None, None, P, 1, 0, None) == INVALID


def test_held_rows_by_hand():
    """The 64-bit form itself, against rows whose codes can be said."""
    y = np.array([[127, -127, 63.5, 0.4, -0.6], [0, 0, 0, 0, 0], [2.0 ** -101, 0, 0, 0, 0], [1, np.inf, 0, 0, 0]], np.float32)
    codes, scales = forms.hold(y)
    assert codes.tolist() == [[127, -127, 64, 0, -1], [0] * 5, [0] * 5, [0] * 5]
    assert scales[0] == 1 and scales[1] == 0 and scales[2] == 0 and np.isnan(scales[3])
