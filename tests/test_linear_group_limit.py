"""grouped_linear takes at most 1024 groups, in the forward as in the backward."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import moe_ops_b200 as M
from moe_ops_b200 import _lib, build


def test_python():
    with FakeTensorMode():
        z = lambda *s, dtype=torch.float32: torch.empty(*s, device="cuda", dtype=dtype)  # noqa: E731
        x = z(3, 8)
        assert M.grouped_linear(x, z(1024, 4, 8), z(1025, dtype=torch.int32)).shape == (3, 4)
        with pytest.raises(ValueError, match="1024"):
            M.grouped_linear(x, z(1025, 4, 8), z(1026, dtype=torch.int32))


def test_c_abi():
    build.build()
    lib, p = _lib.load(), 16
    st = lib.moe_linear_fwd(p, p, p, p, p, None, p, 1026, 3, 4, 8, 1025, 1, 0, 0, p, 1 << 40, None)
    assert st == 1 and b"1024" in lib.moe_last_error_string()
    st = lib.moe_linear_bwd(p, p, p, p, p, p, p, p, 1026, 3, 4, 8, 1025, 1, 4, 0, p, 1 << 40, None)
    assert st == 1 and b"1024" in lib.moe_last_error_string()
