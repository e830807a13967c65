"""The attention over the cache in 8 bits: the workspace that it names (host code: no GPU needed)."""
import pytest


@pytest.fixture(scope="module", params=["bfloat16", "float32"])
def k(request):
    from zse_amd.runtime import build
    from zse_amd.runtime.device import KernelLibrary
    return KernelLibrary(build.ensure("kernels_bf16" if request.param == "bfloat16" else "kernels_f32"), request.param)


def chunk(dtype, table_tokens):
    if dtype == "bfloat16":
        return 256 if table_tokens < 8192 else 512 if table_tokens < 32768 else 1024
    return 128 if table_tokens < 8192 else 256


EDGES = [1, 16, 255, 256, 300, 4000, 8000, 8176, 8190, 8191, 8192, 8193, 16384, 30000, 32752, 32766, 32767, 32768, 32769, 40000, 131072, 1 << 20]


def test_the_largest_call_is_enough_for_the_others(k):
    R, nh, hd = 3, 4, 80
    at = lambda n, w: k.zk_attention_q8_workspace(R, nh, hd, n, w)
    for i, most in enumerate(EDGES):
        for j, widest in enumerate(EDGES[i:], i):
            for n in EDGES[:i + 1]:
                for w in EDGES[:j + 1]:
                    if w >= n:
                        # a partial result: the head's channels filled up to whole 64s, a maximum and a sum
                        assert at(most, widest) >= R * nh * -(-n // chunk(k.dtype, w)) * (128 + 2) * 4, (most, widest, n, w)


def test_no_more_than_the_longest_request_asks_for(k):
    for n, w in ((4000, 4096), (256, 256), (100000, 131072)):
        assert k.zk_attention_q8_workspace(2, 8, 64, n, w) == 2 * 8 * max(-(-min(n, v) // chunk(k.dtype, v)) for v in (8191, 32767, w) if v <= w) * 66 * 4
