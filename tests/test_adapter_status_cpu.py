"""The status word of the adapter's calls is an output like the others: it may not lie in a matrix of
the call (addresses are made up and never followed)."""
import pytest

import xvec_b200 as xb
from test_adapter_cpu import at, gated, gated_backward, linear, linear_backward, refuse


@pytest.mark.parametrize("storage", [1, 2, 3])
@pytest.mark.parametrize("call,inputs,outputs", [
    (linear, (0, 1), (2,)), (gated, (0, 1, 2), (3,)), (linear_backward, (0, 1, 2), (3, 4, 5)),
    (gated_backward, (0, 1, 2, 3, 4, 5), (6, 7, 8, 9, 10))])
def test_status_inside_a_matrix(call, inputs, outputs, storage):
    for i in inputs + outputs:
        refuse(call(storage=storage, status_ptr=at(i) + 4), "overlaps")
    refuse(call(storage=storage, status_ptr=at(0) + 2), "status is not aligned")


def test_status_beside_the_matrices():
    """Directly behind a matrix it is none of its elements: without a device the call then says so."""
    if xb.device_count() > 0:
        pytest.skip("a device is visible: the made-up addresses would be followed")
    for call in (linear, gated, linear_backward, gated_backward):
        with pytest.raises(xb.XvecGPUError) as e:
            call(status_ptr=at(0) + 4 * 4 * 16)()
        assert e.value.status == xb.UNSUPPORTED
