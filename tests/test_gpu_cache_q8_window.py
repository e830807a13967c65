"""Layers whose window is longer than any context, over the cache in 8 bits."""
import numpy as np
import pytest

from gpu_util import make_runner

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_window_up_to_the_largest_number(tmp_path, dtype):
    """Portions, single tokens and both in a step: the bits of a window that is just longer than the longest context."""
    from zse_amd.engine.runner import StepEntry
    from zse_amd.weights import write_random_model
    cfg = dict(architectures=["Gemma2ForCausalLM"], model_type="gemma2", num_hidden_layers=2, hidden_size=64, num_attention_heads=4,
               num_key_value_heads=2, head_dim=32, query_pre_attn_scalar=32, intermediate_size=96, vocab_size=300, rope_theta=10000.0,
               attn_logit_softcapping=30.0, final_logit_softcapping=20.0, rms_norm_eps=1e-6, max_position_embeddings=512)
    tokens = np.random.default_rng(0).integers(0, 300, 200).tolist()
    steps = [[("a", 90)], [("a", 40), ("b", 1)], [("a", 1), ("b", 1)], [("a", 1), ("b", 60)], [("a", 1), ("b", 1)]]
    got = []
    for window in (257, 2 ** 31 - 256, 2 ** 31 - 1):
        folder = write_random_model(str(tmp_path / str(window)), dict(cfg, sliding_window=window), seed=6, std=0.08, gain_std=0.1, dtype=dtype,
                                    std_of={"embed_tokens": 0.02})
        runner = make_runner(folder, dtype, page_size=16, num_pages=40, max_seqs=4, max_batch_tokens=128, max_model_len=256, use_graphs=True,
                             cache_dtype="int8")
        fed, rows = {"a": 0, "b": 7}, []
        for entries in steps:
            rows.append(runner.step([StepEntry(r, tokens[fed[r]:fed[r] + n], list(range(n))) for r, n in entries]))
            for r, n in entries:
                fed[r] += n
        got.append(np.concatenate(rows))
        runner.close()
    assert np.isfinite(got[0]).all() and np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("nh,nkv,hd,bs", [(8, 4, 256, 16), (8, 4, 128, 64), (6, 1, 64, 128), (4, 4, 96, 48), (5, 5, 16, 32)])
def test_portions_behind_a_window_meet_nothing_of_others(tmp_path, nh, nkv, hd, bs, dtype):
    """Portions from 2 to 700 tokens behind a window that begins anywhere in a tile and a page, alone and two in a step: what no request holds, and
    the pages of the compute type before every step, are no numbers, and not a bit moves."""
    from test_gpu_cache_q8_engine import spoil_free_pages
    from zse_amd.engine.runner import StepEntry
    from zse_amd.weights import write_random_model
    cfg = dict(architectures=["Gemma2ForCausalLM"], model_type="gemma2", num_hidden_layers=2, hidden_size=64, num_attention_heads=nh,
               num_key_value_heads=nkv, head_dim=hd, query_pre_attn_scalar=hd, intermediate_size=96, vocab_size=300, rope_theta=10000.0,
               sliding_window=333, rms_norm_eps=1e-6, max_position_embeddings=4096)
    folder = write_random_model(str(tmp_path / "m"), cfg, seed=6, std=0.08, gain_std=0.1, dtype=dtype, std_of={"embed_tokens": 0.02})
    rng = np.random.default_rng(hd)
    streams = {"a": rng.integers(0, 300, 2600).tolist(), "b": rng.integers(0, 300, 1200).tolist()}
    steps = [[("a", 700)], [("a", 513), ("b", 450)], [("a", 2), ("b", 33)], [("a", 64), ("b", 1)], [("b", 257)], [("a", 700), ("b", 17)], [("a", 1), ("b", 3)]]

    def run(spoiled):
        runner = make_runner(folder, dtype, page_size=bs, cache_tokens=4096, max_seqs=3, max_batch_tokens=1024, max_model_len=2600, use_graphs=False,
                             cache_dtype="int8")
        fed, rows = {r: 0 for r in streams}, []
        for entries in steps:
            if spoiled:
                spoil_free_pages(runner)
            rows.append(runner.step([StepEntry(r, streams[r][fed[r]:fed[r] + n], [0, n - 1]) for r, n in entries]))
            for r, n in entries:
                fed[r] += n
        runner.close()
        return np.concatenate(rows)

    clean, dirty = run(False), run(True)
    assert np.isfinite(clean).all() and np.array_equal(clean, dirty)
