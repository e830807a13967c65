"""The cache in 8 bits: further calls that are refused (host code: no GPU needed)."""
import pytest

from test_cache_q8 import A, ATTEND, WRITE, k  # noqa: F401  (a fixture)


# three rows of 8 + 2 x 4 heads of 128: two planes are 3 * 2,048 * 4 bytes each, three rows of queries 2 * ldq + 1,024 values
@pytest.mark.parametrize("q_out", [A, A + 16, A + 2 * 3 * 2048 * 4 - 16, A - 16])
@pytest.mark.parametrize("ldq", [1024, 2048])
def test_queries_over_the_partial_sums(k, q_out, ldq):
    from zse_amd.runtime.device import DeviceError
    with pytest.raises(DeviceError, match="zk_rope_cache_write_q8.*queries over the partial sums"):
        k.zk_rope_cache_write_q8(*dict(WRITE, qkv=None, ld=0, planes=A, sums=2, q_out=q_out, ldq=ldq).values())


@pytest.mark.parametrize("cap", [float("inf"), float("nan"), float("-inf")])
def test_caps_that_are_no_numbers(k, cap):
    """An infinite cap is infinity times the tangent of zero: no number, where a caller may have meant no cap."""
    from zse_amd.runtime.device import DeviceError
    with pytest.raises(DeviceError, match="zk_attention_q8.*softcap must be finite"):
        k.zk_attention_q8(*dict(ATTEND, softcap=cap).values())
