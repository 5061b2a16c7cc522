"""The torch operators' library runs on torch's own C++ runtime."""

from rational_kat_cu_b200 import _build


def test_one_cpp_runtime():
    """A static copy of libstdc++ beside torch's crashed where an error message held a number."""
    with open(_build.build_torch(), "rb") as f:
        assert b"\0libstdc++.so.6\0" in f.read()
