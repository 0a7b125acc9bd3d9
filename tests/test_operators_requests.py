"""More of what the operators' entry points refuse before they touch a device."""
import pytest

from poorgrad_b200 import abi
from test_operators_host import INVALID, policy_request, preference_request, scan_request


@pytest.mark.parametrize("entry,request_bytes", [
    ("tb_gated_scan", scan_request(clear=8)), ("tb_gated_scan", scan_request(clear=-1)),
    ("tb_gated_scan_backward", scan_request(clear=1 << 40)),
    ("tb_preference_loss", preference_request(clear=4)), ("tb_preference_loss", preference_request(clear=-2))])
def test_only_known_arrays_are_cleared(built, entry, request_bytes):
    lib = abi.load_library()
    assert getattr(lib, entry)(request_bytes, None) == INVALID
    assert b"clear" in lib.tb_last_error()


@pytest.mark.parametrize("scale", [2.5e38, 2.9e38, 1e300, float("inf")])
def test_a_scale_past_what_the_exponentials_take(built, scale):
    """scale log2(e) is what logits are multiplied by: an infinite one would make NaN of every row."""
    lib = abi.load_library()
    assert lib.tb_policy_loss(policy_request(scale=scale), None) == INVALID
    assert lib.tb_preference_loss(preference_request(scale=scale), None) == INVALID
    assert lib.tb_token_logp(0, 256, 5, 256, 2, 5, scale, 256, None) == INVALID
    assert b"scale" in lib.tb_last_error()
