"""Which C entries take a dense product as offsets NULL, num_offsets 0, one expert: moe_gmm_fwd, _dgrad
and _wgrad and the linear ones (documented so); the others refuse it, as they did before."""
import pytest

from moe_ops_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def test_refused(lib):
    p, sizes = 16, (4, 8, 8)
    calls = {
        "moe_gmm_fwd_gather": (p, p, 4, p, p, None, 0, *sizes, 1, 1, 2, None),
        "moe_gmm_wgrad_gather": (p, p, 4, p, p, None, 0, *sizes, 1, 1, 2, None),
        "moe_gmm_dgrad_dual": (p, p, p, p, p, None, 0, 4, 8, 8, 8, 1, 1, 2, None),
        "moe_gmm_gate_up_fwd": (p, p, p, p, p, p, None, 0, *sizes, 1, 1, 2, None),
        "moe_gmm_gate_up_fwd_gather": (p, p, 4, p, p, p, p, p, None, 0, *sizes, 1, 1, 2, None),
        "moe_gmm_dgrad_swiglu_bwd": (p, p, p, p, p, p, None, 0, *sizes, 1, 1, 2, None),
    }
    for name, args in calls.items():
        assert getattr(lib, name)(*args) == 1, name
        assert b"num_offsets" in lib.moe_last_error_string(), name


def test_taken(lib):
    p = 16
    for name in ("moe_gmm_fwd", "moe_gmm_dgrad", "moe_gmm_wgrad"):
        # past the checks of the arguments: no rows, nothing to launch
        assert getattr(lib, name)(p, p, p, None, 0, 0, 8, 0, 1, 1, 2, None) != 1, name
