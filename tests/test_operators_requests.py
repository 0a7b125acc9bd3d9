"""More of what the operators' entry points refuse before they touch a device."""
import pytest

from poorgrad_b200 import abi
from test_operators_host import INVALID, preference_request, scan_request


@pytest.mark.parametrize("entry,request_bytes", [
    ("tb_gated_scan", scan_request(clear=8)), ("tb_gated_scan", scan_request(clear=-1)),
    ("tb_gated_scan_backward", scan_request(clear=1 << 40)),
    ("tb_preference_loss", preference_request(clear=4)), ("tb_preference_loss", preference_request(clear=-2))])
def test_only_known_arrays_are_cleared(built, entry, request_bytes):
    lib = abi.load_library()
    assert getattr(lib, entry)(request_bytes, None) == INVALID
    assert b"clear" in lib.tb_last_error()
