"""What the library gives to the process that loads it: its C entry points, and no name that another library could share with it."""
import shutil
import subprocess

import pytest

from diffgemma_b200 import capi


@pytest.mark.skipif(shutil.which("nm") is None, reason="needs nm")
def test_no_common_names_are_exported():
    capi.load()
    lines = subprocess.run(["nm", "-D", "--defined-only", capi.LIB_PATH], capture_output=True, text=True, check=True).stdout.splitlines()
    names = [(x.split()[-2], x.split()[-1]) for x in lines]
    assert any(n == "dg_last_error_message" for _, n in names)
    # unique symbols are one for the whole process, and keep the library from being unloaded
    assert [n for t, n in names if t == "u"] == []
    # functions outside a namespace, but for the standard library's templates and the compiler's stubs of kernels
    assert [n for _, n in names if n.startswith("_Z") and not n.startswith(("_ZN", "_ZSt")) and "__device_stub__" not in n] == []
