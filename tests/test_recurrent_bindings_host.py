"""Host-only checks of what the bindings of the recurrent operators make of arguments that are left
out."""
import os
import re

import numpy as np
import pytest

from ilgpu_amd import capi
from tests.test_recurrent_operators_host import host_array


def test_an_input_weight_stands_for_an_input_norm_in_the_gradients_too():
    # The forward call takes it so; its gradients need input_rstd then, and say so before any GPU work.
    f32 = np.float32
    x = capi.DeviceMatrix(host_array(24, f32), 6, 4)
    args = dict(grad_out=None, grad_total=x, inp=x, total=None, weight=None, rstd=None, grad_in=x, stream=0,
                temp=host_array(1 << 16, np.int32), input_weight=host_array(4, f32))
    with pytest.raises(capi.ArgumentNullError):
        capi.residual_norm_gradient(**args)
    with pytest.raises(capi.ArgumentNullError):
        capi.residual_norm_gradient(**args, input_norm=True)
    none = capi.DeviceMatrix(host_array(0, f32), 0, 4)
    capi.residual_norm_gradient(**{**args, "grad_total": none, "inp": none, "grad_in": none})


def test_a_default_block_output_of_the_csharp_layer_is_passed_on_as_it_is():
    # A struct is all zeros unless its constructor is called: what has another value where nothing was set
    # is no plain field.  The C ABI's scale is 1, and the other layers' gate is silu.
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "csharp",
                        "ILGPU.Algorithms.Hip", "HipRecurrentModelExtensions.cs")
    text = open(path).read()
    struct = text[text.index("public struct HipBlockOutput"):]
    struct = struct[:struct.index("\n    }\n")]
    assert re.search(r"private float\? scale;", struct) and re.search(r"private HipGateKind\? kind;", struct)
    for kind, name, value in (("float", "Scale", "scale ?? 1.0f"), ("HipGateKind", "Kind", "kind ?? HipGateKind.Silu")):
        assert not re.search(rf"public {kind} {name};", struct)
        body = re.search(rf"public {kind} {name}\s*{{(.*?)\n        }}", struct, flags=re.S)[1]
        assert f"get => {value};" in body and "set => " in body
