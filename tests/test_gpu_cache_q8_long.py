"""Attention over the cache in 8 bits where a request meets more chunks of keys than a wave has lanes, against float64."""
import numpy as np
import pytest

from plain import cache_q8_plain as P

pytestmark = pytest.mark.gpu

HALF = {"bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}      # half a step of a rounding, relative to the value
CHUNK = {"bfloat16": 1024, "float32": 256}                 # keys of a partial result in tables as wide as these


@pytest.fixture(scope="module")
def rt():
    from zse_amd.runtime.device import Runtime
    return Runtime.get()


def rounded(x, dtype):
    from zse_amd.weights.safetensors import bf16_bits_to_f32, f32_to_bf16_bits
    x = np.ascontiguousarray(x, np.float32)
    return bf16_bits_to_f32(f32_to_bf16_bits(x)).reshape(x.shape) if dtype == "bfloat16" else x


def up(rt, x, dtype):
    from zse_amd.weights.safetensors import f32_to_bf16_bits
    x = np.ascontiguousarray(x, np.float32)
    return rt.upload(f32_to_bf16_bits(x), "bfloat16") if dtype == "bfloat16" else rt.upload(x)


def cached(codes, scales, pages, head, hd, form, values):
    """[tokens, hd] of a head's pages in their order, by the layout's definition."""
    x = P.numbers(np.arange(256), form)[codes[pages, head]]                        # [pages, pieces, blocks, 1024]
    n, pieces, blocks, _ = x.shape
    if values:
        x = x.reshape(n, pieces, blocks, 4, 16, 4, 4).transpose(0, 1, 3, 6, 2, 5, 4)     # .. token 4 a + d, block, channel 16 c + b
    else:
        x = x.reshape(n, pieces, blocks, 16, 64).transpose(0, 1, 3, 2, 4)
    x = x.reshape(n * pieces * 16, blocks * 64)[:, :hd]
    return x * scales[pages, head, int(values)].reshape(-1, 1).astype(np.float64)


@pytest.mark.parametrize("chunks,window", [(64, False), (65, False), (65, True), (128, False), (129, True), (150, False)])
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 64), (3, 1, 40), (2, 1, 128), (2, 1, 192), (2, 1, 256)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_more_chunks_than_lanes(rt, dtype, nh, nkv, hd, chunks, window):
    """A long request beside a short one; the window begins inside a chunk and meets as many chunks as are asked for."""
    rng = np.random.default_rng(chunks + hd)
    k, bs, form, chunk = rt.kernels(dtype), 128, chunks % 2, CHUNK[dtype]
    before = 2 * chunk + 100 if window else 0              # positions in front of the window
    n, short = before // chunk * chunk + chunks * chunk - 37, 300
    used = [-(-n // bs), -(-short // bs)]
    width, pages = max(used[0], (32768 if dtype == "bfloat16" else 8192) // bs), sum(used) + 1
    ids = 1 + rng.permutation(pages - 1)
    table = np.full((2, width), -1, np.int32)
    table[0, :used[0]], table[1, :used[1]] = ids[:used[0]], ids[used[0]:]
    codes = [rng.integers(0, 252, (pages, nkv, bs // 16, -(-hd // 64), 1024), dtype=np.uint8) for _ in range(2)]
    for x in codes:
        x += np.where(x < 126, np.uint8(1), np.uint8(3))                           # (none of 0x00, 0x7f, 0x80 and 0xff)
    scales = (np.exp(rng.standard_normal((pages, nkv, 2, bs)) * 0.4) / P.TOP[form]).astype(np.float32)
    q = rounded(rng.standard_normal((2, nh, hd)), dtype)
    # scores of a standard deviation of about four: the chunks' maxima differ, and what each of them is worth matters
    scale = 4 / (np.sqrt(hd) * np.sqrt(np.mean(P.numbers(codes[0][1], form) ** 2)) / P.TOP[form])
    lens, win = [n, short], n - before if window else 0
    assert -(-n // chunk) - before // chunk == chunks
    Q, TBL, CL = up(rt, q.reshape(2, -1), dtype), rt.upload(table), rt.upload(np.array(lens, np.int32))
    KC, VC, SC = rt.upload(codes[0]), rt.upload(codes[1]), rt.upload(scales)
    room = k.zk_attention_q8_workspace(2, nh, hd, n, width * bs)
    WS, OUT = rt.upload(np.full((room // 4 + 1,), np.nan, np.float32)), up(rt, np.full((2, nh * hd), 5.0), dtype)
    k.zk_attention_q8(Q.ptr, nh * hd, KC.ptr, VC.ptr, SC.ptr, TBL.ptr, width, CL.ptr, OUT.ptr, 2, n, nh, nkv, hd, bs, pages, float(scale),
                      0.0, win, form, WS.ptr, room, rt.stream)
    got = rt.download_f32(OUT).reshape(2, nh, hd)
    scale = np.float64(np.float32(scale))
    for r, m in enumerate(lens):
        first = max(0, m - win) if win else 0
        for g in range(nkv):
            keys, values = (cached(x, scales, table[r, :used[r]], g, hd, form, bool(v))[first:m] for v, x in enumerate(codes))
            for h in range(g * (nh // nkv), (g + 1) * (nh // nkv)):
                x = q[r, h].astype(np.float64)
                z = keys @ x * scale
                p = np.exp(z - z.max())
                p /= p.sum()
                want, spread = p @ values, p @ np.abs(values)
                # A score is off by hd roundings of its sum of |q| |k| and by eight of its own factors.  A weight is off by twice that,
                # by its rounding (24 bits, or 16 as two numbers) and by an exponential's two steps, twice where a chunk is joined.  A
                # sum has at most a chunk's keys in a chain, the other waves and then the chunks.
                score = (np.abs(keys) @ np.abs(x)).max() * scale * (hd + 8) * 2.0 ** -24
                weight = (2.0 ** -16 if dtype == "bfloat16" else 0.0) + (chunk + chunks + 64) * 2.0 ** -23
                tol = spread * (2 * score + weight) + np.abs(want) * HALF[dtype] * 1.01
                assert (np.abs(got[r, h] - want) <= tol).all(), (r, h, np.abs(got[r, h] - want).max(), tol.min(), np.abs(want).max())
