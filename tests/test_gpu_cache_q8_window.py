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
