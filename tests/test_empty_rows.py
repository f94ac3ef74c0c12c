"""Row operands that hold no element: their strides address nothing, so none is
refused, also where those of a batch with elements would be. The host checks run
without a device; the weights' gradients over no rows are zeros."""
import ctypes

import numpy as np
import pytest

import chelis_amd as C
from block_reference import NP, encode
from test_block_refusals import BF16, EUNSUPPORTED, F32, ref, refused, tensor

# (shape, strides): leading axes that do not collapse, a last axis with a step
EMPTY = [((2, 0, 16), (1000, 7, 1)), ((3, 4, 0, 16), (1000, 7, 5, 1)), ((0, 16), (40, 2)), ((2, 0, 16), (32, 1, 2))]


def accepted(status):
    assert status == 0, C.lib().chelis_hip_last_error().decode()


@pytest.mark.parametrize("shape,strides", EMPTY)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_forward_calls(shape, strides, dtype):
    x, y = tensor(shape, dtype, strides), tensor(shape, dtype)
    w, stat = lambda: tensor((16,), dtype), lambda: tensor(shape[:-1], F32)
    lib = C.lib()
    accepted(lib.chelis_hip_layer_norm_stats(ref(x), ref(w()), ref(w()), 1e-5, ref(y), ref(stat()), ref(stat())))
    side = C.NormSide(2, 0, ctypes.pointer(w()), None, None, ctypes.pointer(stat()))
    accepted(lib.chelis_hip_residual_norm(ref(x), ref(tensor(shape, dtype)), None, None, 0.5, ctypes.byref(side), 1e-5,
                                          ref(y), ref(tensor(shape, dtype))))
    if dtype == BF16:
        m = tensor((16, 24), dtype)
        accepted(lib.chelis_hip_dense(ref(x), ref(m), None, 0, None, ref(tensor(shape[:-1] + (24,), dtype)), None))


def test_the_same_strides_with_elements_are_refused():
    x = tensor((2, 3, 16), F32, (1000, 20, 1))
    refused(C.lib().chelis_hip_layer_norm_stats(ref(x), ref(tensor((16,))), ref(tensor((16,))), 1e-5, ref(tensor((2, 3, 16))),
                                                ref(tensor((2, 3))), ref(tensor((2, 3)))), "uniform row stride", EUNSUPPORTED)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("shape,strides", EMPTY)
def test_weight_gradients_are_zeros(kind, shape, strides):
    n = shape[-1]
    ones = lambda *s: C.to_device(encode(kind, np.ones(s)))
    x = C.empty((4000,), NP[kind]).view(shape, strides)
    stat = lambda: C.empty(shape[:-1], np.float32)
    dx, dgamma, dbeta = C.layer_norm_adjoint(x, ones(n), stat(), stat(), x, C.empty(shape, NP[kind]), ones(n), ones(n))
    assert dx.shape == shape and not dgamma.numpy().any() and not dbeta.numpy().any()
    norm = C.Norm("layer", ones(n), ones(n), stat(), stat())
    _, _, _, _, dpre = C.residual_norm_adjoint(x, pre=norm, dh=x, dx=C.empty(shape, NP[kind]), dpre=(ones(n), ones(n)))
    assert not dpre[0].numpy().any() and not dpre[1].numpy().any()
