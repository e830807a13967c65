"""The cache in 8 bits: what its entry points refuse, and the sizes they name (host code: no GPU needed)."""
import ctypes as C

import numpy as np
import pytest

from plain import cache_q8_plain as P


@pytest.fixture(scope="module", params=["bfloat16", "float32"])
def k(request):
    from zse_amd.runtime import build
    from zse_amd.runtime.device import KernelLibrary
    return KernelLibrary(build.ensure("kernels_bf16" if request.param == "bfloat16" else "kernels_f32"), request.param)


A = 4096            # an address that is never read: every call below ends before a launch

WRITE = dict(qkv=A, ld=2048, planes=None, sums=0, q_out=A, ldq=2048, positions=A, slot_map=A, inv_freq=A, rotary_dim=128, kcodes=A, vcodes=A,
             scales=A, T=3, nh=8, nkv=4, hd=128, bs=16, num_pages=9, format=0, stream=None)
READ = dict(kcodes=A, vcodes=A, scales=A, block_table=A, max_blocks=8, q_start=None, ctx_len=A, k=A, v=A, R=2, max_ctx=128, window=0, nkv=4, hd=128,
            bs=16, num_pages=9, v_transposed=1, format=1, stream=None)
ATTEND = dict(q=A, q_stride=1024, kcodes=A, vcodes=A, scales=A, block_table=A, max_blocks=8, ctx_len=A, out=1 << 30, R=2, max_ctx=128, nh=8, nkv=4, hd=128,
              bs=16, num_pages=9, scale=0.1, softcap=0.0, window=0, format=0, workspace=A, workspace_bytes=1 << 30, stream=None)

CACHE = [(dict(bs=8), "pages of 16"), (dict(bs=0), "pages of 16"), (dict(bs=24), "pages of 16"), (dict(num_pages=0), "one page"),
         (dict(hd=257), "256 channels"), (dict(bs=1 << 23), "2 GiB"), (dict(hd=0), ""), (dict(format=2), "format"), (dict(format=-1), "format"), (dict(kcodes=A + 8), "16"),
         (dict(vcodes=None), "16"), (dict(scales=A + 4), "16")]


@pytest.mark.parametrize("change,says", CACHE + [
    (dict(T=-1), "bad sizes"), (dict(nh=0), "bad sizes"), (dict(nkv=-1), "bad sizes"), (dict(sums=-1), "bad sizes"), (dict(nkv=20000), "too many"),
    (dict(rotary_dim=3), "even"), (dict(rotary_dim=130), "at most"), (dict(inv_freq=None), "frequency"), (dict(ld=2047), "overlap"),
    (dict(ldq=1023), "overlap"), (dict(qkv=None), "null"), (dict(q_out=None), "null"), (dict(positions=None), "null"),
    (dict(sums=2, planes=None), "null"), (dict(sums=2, planes=A + 4), "misaligned"),
    (dict(ldq=1024, q_out=A), "where they came from"), (dict(q_out=A + 64, ldq=2048), "where they came from")])
def test_write_refuses(k, change, says):
    from zse_amd.runtime.device import DeviceError
    with pytest.raises(DeviceError, match=f"zk_rope_cache_write_q8.*{says}"):
        k.zk_rope_cache_write_q8(*dict(WRITE, **change).values())


@pytest.mark.parametrize("change,says", CACHE + [
    (dict(R=-1), "bad sizes"), (dict(max_ctx=-1), "bad sizes"), (dict(window=-1), "bad sizes"), (dict(max_ctx=129), "longer than the table"),
    (dict(max_ctx=2 ** 30 + 1, max_blocks=2 ** 30), "2\\^30"), (dict(nkv=0), ""), (dict(nkv=70000), "too many"), (dict(R=70000), "too many"), (dict(block_table=None), "null"), (dict(ctx_len=None), "null"),
    (dict(k=None), "null"), (dict(v=A + 8), "misaligned")])
def test_read_refuses(k, change, says):
    from zse_amd.runtime.device import DeviceError
    with pytest.raises(DeviceError, match=f"zk_cache_read_q8.*{says}"):
        k.zk_cache_read_q8(*dict(READ, **change).values())


@pytest.mark.parametrize("change,says", CACHE + [
    (dict(R=-1), "bad sizes"), (dict(max_ctx=-5), "bad sizes"), (dict(window=-1), "bad sizes"), (dict(nh=0), "bad sizes"),
    (dict(nh=9), "multiple"), (dict(q_stride=1023), "overlap"), (dict(nh=70000, q_stride=70000 * 128), "too many"),
    (dict(max_ctx=129), "longer than the table"), (dict(softcap=-1.0), "softcap"), (dict(q=None), "null"), (dict(out=None), "null"),
    (dict(ctx_len=None), "null"), (dict(block_table=None), "null"), (dict(R=70000), "too many"), (dict(num_pages=1 << 30), "too many pages"),
    (dict(max_ctx=2 ** 30 + 1, max_blocks=2 ** 30), "2\\^30"), (dict(max_ctx=2 ** 30, max_blocks=2 ** 30), "too many chunks"),
    (dict(out=A + 2 * 1024), "results over queries"), (dict(max_ctx=20000, max_blocks=2000, workspace=None), "no workspace"), (dict(max_ctx=20000, max_blocks=2000, workspace=A + 4), "multiple of 16"),
    (dict(max_ctx=20000, max_blocks=2000, workspace_bytes=1000), "too small")])
def test_attention_refuses(k, change, says):
    from zse_amd.runtime.device import DeviceError
    with pytest.raises(DeviceError, match=f"zk_attention_q8.*{says}"):
        k.zk_attention_q8(*dict(ATTEND, **change).values())


def test_nothing_to_do(k):
    k.zk_rope_cache_write_q8(*dict(WRITE, T=0).values())
    k.zk_cache_read_q8(*dict(READ, R=0).values())
    k.zk_cache_read_q8(*dict(READ, max_ctx=0).values())
    k.zk_attention_q8(*dict(ATTEND, R=0).values())


def test_calls_can_be_written_down(k):
    for name in ("zk_rope_cache_write_q8", "zk_cache_read_q8", "zk_attention_q8"):
        assert k._dll.zk_steplist_op(name.encode()) >= 0


def test_bytes(k):
    assert k.zk_cache_q8_bytes(3, 4, 128, 16) == 3 * 4 * 128 * 16
    assert k.zk_cache_q8_bytes(3, 5, 80, 32) == 3 * 5 * 128 * 32          # the last block of channels is filled up
    assert k.zk_cache_q8_bytes(1 << 20, 16, 256, 128) == (1 << 20) * 16 * 256 * 128
    for bad in ((0, 4, 128, 16), (3, 0, 128, 16), (3, 4, 0, 16), (3, 4, 257, 16), (3, 4, 128, 20)):
        assert k.zk_cache_q8_bytes(*bad) == 0


def test_workspace(k):
    most = k.zk_attention_q8_workspace(64, 8, 128, 8192, 8192)
    assert most > 0
    for less in ((63, 8, 128, 8192, 8192), (64, 8, 128, 4000, 8192), (64, 7, 128, 8192, 8192), (64, 8, 64, 8192, 8192)):
        assert k.zk_attention_q8_workspace(*less) < most
    for none in ((0, 8, 128, 8192, 8192), (64, 0, 128, 8192, 8192), (64, 8, 257, 8192, 8192), (64, 8, 128, 0, 8192)):
        assert k.zk_attention_q8_workspace(*none) == 0


def test_layout_is_one_to_one():
    for hd in (64, 80, 256):
        c = P.Cache(1, 1, hd, 32, 0)
        for values in (False, True):
            seen = set()
            for off in range(32):
                block, at = c.places(off, values)
                seen |= {(off // 16, int(b), int(a)) for b, a in zip(block, at)}
            assert len(seen) == 32 * hd and max(a for _, _, a in seen) < 1024


def test_numbers():
    assert P.numbers(np.array([0x7e, 0xfe, 0x38, 0x01, 0x00], np.uint8), 1).tolist() == [448.0, -448.0, 1.0, 2.0 ** -9, 0.0]
    assert P.numbers(np.array([0x7f, 0x81, 0xff, 0], np.uint8), 0).tolist() == [127.0, -127.0, -1.0, 0.0]


def test_names():
    from zse_amd.runtime.device import canonical_cache_dtype
    assert canonical_cache_dtype(None, "bfloat16") is None and canonical_cache_dtype("bf16", "bfloat16") is None
    assert canonical_cache_dtype("float32", "fp32") is None
    assert canonical_cache_dtype("INT8", "float32") == "int8" and canonical_cache_dtype("fp8", "bfloat16") == "float8_e4m3"
    for bad in ("int4", "float32", ""):
        with pytest.raises(ValueError, match="cache_dtype must be one of"):
            canonical_cache_dtype(bad, "bfloat16")
