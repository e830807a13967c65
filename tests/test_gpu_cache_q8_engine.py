"""The engine over a cache in 8 bits: steps of every kind against a float64 run that rounds keys and values likewise, graphs, launch
lists and batches bit for bit, windows, preemption, what is refused."""
import numpy as np
import pytest

from conftest import TINY, read_weights
from gpu_util import BF16_REL, F32_ATOL, bf16_round, make_runner, run_steps
from plain import cache_q8_plain as Q
from plain import gemma2_plain as P

pytestmark = pytest.mark.gpu

FORMATS = {"int8": 0, "float8_e4m3": 1}


def held(x, form):
    """[T, heads, hd] as a cache of this format holds it."""
    top = Q.TOP[form]
    a = np.abs(x).max(axis=-1, keepdims=True)
    scale = a / top
    code = x / np.where(scale == 0, 1, scale)
    if form == 0:
        return np.round(code) * scale
    numbers = np.unique(Q.numbers(np.arange(256, dtype=np.uint8), 1)[~np.isnan(Q.numbers(np.arange(256, dtype=np.uint8), 1))])
    return numbers[np.searchsorted((numbers[1:] + numbers[:-1]) / 2, code)] * scale


def reference(monkeypatch, name, dtype, folder, tokens, form):
    """Float64 logits, keys and values rounded to the format (form None: as they are)."""
    H = TINY[name][0]["hidden_size"]
    scale = np.float64(np.float32(np.sqrt(H))) if dtype == "float32" else np.float64(bf16_round(np.sqrt(H)))
    plain = P.attention
    with monkeypatch.context() as m:
        if form is not None:
            m.setattr(P, "attention", lambda q, k, v, *a: plain(q, held(k, form), held(v, form), *a))
        return P.forward(TINY[name][0], read_weights(folder), tokens, np.float64, embed_scale=scale)


CUTS = {"whole": [60], "portions": [17, 1, 30, 12], "single": [1] * 60, "mixed": [33] + [1] * 20 + [7]}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("cache_dtype", ["int8", "float8_e4m3"])
@pytest.mark.parametrize("name", ["A", "B"])
def test_steps_of_every_kind(monkeypatch, tiny_folders, name, cache_dtype, dtype):
    folder = tiny_folders[(name, dtype)]
    rng = np.random.default_rng(3)
    tokens = rng.integers(0, TINY[name][0]["vocab_size"], 60).tolist()
    want = reference(monkeypatch, name, dtype, folder, tokens, FORMATS[cache_dtype])
    rounding = np.abs(want - reference(monkeypatch, name, dtype, folder, tokens, None)).max()
    assert rounding > 0
    for cut, sizes in CUTS.items():
        runner = make_runner(folder, dtype, page_size=16, num_pages=16, max_seqs=4, max_batch_tokens=128, max_model_len=256, use_graphs=True,
                             cache_dtype=cache_dtype)
        # a second request beside, single tokens and a portion
        other = rng.integers(0, TINY[name][0]["vocab_size"], len(sizes) + 4).tolist()
        steps = [([("r", n), ("o", 5 if i == 0 else 1)], []) for i, n in enumerate(sizes)]
        got = run_steps(runner, {"r": tokens, "o": other}, steps)["r"]
        err = np.abs(got - want)
        if dtype == "float32":
            # Sums in another order move a value of 2^-23 or so across a code's border now and then; that changes one value by a code's step,
            # where the rounding of all of them, by up to half a step each, changes the logits by ``rounding``.
            assert err.max() < rounding / 4 + F32_ATOL and np.median(err) < F32_ATOL, (cut, err.max(), rounding)
        else:
            # A value that is off by d before it is held is held as one at most d and two half steps away from the reference's (half a
            # step on either side), where ``rounding`` is what one half step at the most does: what 16 bits may be off by, and twice that.
            assert err.max() < BF16_REL * np.abs(want).max() + 2 * rounding, (cut, err.max(), np.abs(want).max(), rounding)
        runner.close()


def decode(runner, prompts, steps):
    """Greedy rows: prompts in one step, then single tokens; the first request's rows."""
    from zse_amd.engine.runner import StepEntry
    rows, toks = [], {}
    z = runner.step([StepEntry(i, p, [len(p) - 1]) for i, p in enumerate(prompts)])
    for s in range(steps):
        rows.append(z[0].copy())
        toks = [int(np.argmax(z[i])) for i in range(len(prompts))]
        z = runner.step([StepEntry(i, [t], [0]) for i, t in enumerate(toks)])
    return np.stack(rows)


@pytest.mark.parametrize("cache_dtype", ["int8", "float8_e4m3"])
def test_graphs_lists_and_batches_give_the_same_bits(tiny_folders, cache_dtype):
    folder = tiny_folders[("B", "bfloat16")]
    rng = np.random.default_rng(8)
    prompts = [rng.integers(0, 1000, n).tolist() for n in (50, 33, 7, 90, 1, 16, 17)]
    kw = dict(page_size=16, num_pages=200, max_seqs=8, max_batch_tokens=512, max_model_len=512, cache_dtype=cache_dtype)

    def run(many, **more):
        runner = make_runner(folder, "bfloat16", **dict(kw, **more))
        first = decode(runner, prompts[:1], 1)          # the prompt alone: its rows do not follow from the others'
        runner.finish(0)
        from zse_amd.engine.runner import StepEntry
        for i, p in enumerate(prompts[:many]):
            z = runner.step([StepEntry(i, p, [len(p) - 1])])
        rows, tok = [], [5] * many
        for s in range(12):
            z = runner.step([StepEntry(i, [t], [0]) for i, t in enumerate(tok)])
            rows.append(z[0].copy())
            tok = [int(np.argmax(z[0]))] * many
        stats = (runner.graph_runs, runner.steplist_runs)
        runner.close()
        return np.concatenate([first, np.stack(rows)]), stats

    eager, s = run(1, use_graphs=False, use_steplists=False)
    assert s == (0, 0)
    lists, s = run(1, use_graphs=False)
    assert s[1] > 0
    graphs, s = run(1, use_graphs=True)
    assert s[0] > 0
    beside, s = run(7, use_graphs=True)
    assert s[0] > 0
    assert np.array_equal(eager, lists) and np.array_equal(eager, graphs) and np.array_equal(eager, beside)


def spoil_free_pages(runner):
    """What no request holds, and all that lies behind a request's last token: codes and scales that are no numbers."""
    from zse_amd.runtime.device import Tensor
    rt, m = runner.rt, runner.manager
    bs = runner.page_size
    for c in runner.caches:
        pages, free = c.k.shape[0], None
        free = np.ones(pages, bool)
        free[0] = False
        used = np.zeros((pages, bs), bool)
        for req in list(m._reqs):
            table = m._reqs[req].tables[c.group]
            for j, p in enumerate(table):
                if p > 0:
                    free[p] = False
                    used[p, :max(0, min(bs, m.computed(req) - j * bs))] = True
        nkv = c.scales.shape[1]
        for t, values in ((c.k, False), (c.v, True)):
            whole = rt.download(t).reshape(pages, nkv, bs // 16, -1, 1024)
            at = np.arange(1024)
            token = at // 256 * 4 + at % 4 if values else at // 64
            gone = ~used.reshape(pages, 1, bs // 16, 1, 16)[..., token]
            gone[0] = False
            rt.copy_h2d(t.ptr, np.where(gone, np.uint8(0x7f), whole))
        scales = rt.download(c.scales)
        keep = used[:, None, None, :] | (np.arange(pages) == 0)[:, None, None, None]
        rt.copy_h2d(c.scales.ptr, np.where(keep, scales, np.float32(np.nan)))
        for t in (c.work_k, c.work_v):
            x = rt.download(t)
            x[1:] = 0x7fc0 if t.dtype == "bfloat16" else np.nan
            rt.copy_h2d(t.ptr, x)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_what_others_left_never_reaches_a_request(tmp_path, dtype):
    """As the test of the same name over the compute type's pages: a portion behind 836 tokens, windows with holes, pages handed on."""
    from zse_amd.engine.runner import StepEntry
    from zse_amd.weights import write_random_model
    cfg = dict(architectures=["Gemma2ForCausalLM"], model_type="gemma2", num_hidden_layers=2, hidden_size=64, num_attention_heads=4,
               num_key_value_heads=2, head_dim=32, query_pre_attn_scalar=32, intermediate_size=96, vocab_size=300, rope_theta=10000.0,
               sliding_window=200, attn_logit_softcapping=30.0, final_logit_softcapping=20.0, rms_norm_eps=1e-6, max_position_embeddings=4096)
    folder = write_random_model(str(tmp_path / "m"), cfg, seed=6, std=0.08, gain_std=0.1, dtype=dtype, std_of={"embed_tokens": 0.02})
    rng = np.random.default_rng(4)
    streams = {"long": rng.integers(0, 300, 960).tolist(), "short": rng.integers(0, 300, 301).tolist(), "late": rng.integers(0, 300, 77).tolist()}
    steps = [([("long", 836)], []), ([("long", 64), ("short", 289)], []), ([("long", 40), ("short", 1)], [])]
    steps += [([("long", 1), ("short", 1)], []) for _ in range(5)] + [([("long", 1), ("short", 1)], ["short"])]
    steps += [([("long", 1), ("late", 33)], []), ([("long", 1), ("late", 44)], ["late"])] + [([("long", 1)], []) for _ in range(12)]

    def run(spoiled):
        runner = make_runner(folder, dtype, page_size=16, num_pages=90, max_seqs=4, max_batch_tokens=1024, max_model_len=4096, use_graphs=True,
                             cache_dtype="float8_e4m3")
        fed, rows = {r: 0 for r in streams}, []
        for entries, ends in steps:
            if spoiled:
                spoil_free_pages(runner)
            rows.append(runner.step([StepEntry(r, streams[r][fed[r]:fed[r] + n], [n - 1]) for r, n in entries]))
            for r, n in entries:
                fed[r] += n
            for r in ends:
                runner.finish(r)
        runner.close()
        return np.concatenate(rows)

    clean, dirty = run(False), run(True)
    assert np.isfinite(clean).all() and np.array_equal(clean, dirty)


@pytest.mark.parametrize("cache_dtype", ["int8", "float8_e4m3"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generate(tiny_folders, dtype, cache_dtype):
    """Through the engine: prompts in portions beside decoded tokens, few pages (requests give theirs up and start again), the same ids as
    with room for everybody where the two runs cut the prompts alike."""
    from zse_amd.engine.engine import Engine
    from zse_amd.sampling import SamplingParams
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, 512, n).tolist() for n in (5, 70, 33, 16, 1, 100)]
    outs = []
    for blocks, seqs in ((64, 6), (14, 6)):
        eng = Engine(tiny_folders[("A", dtype)], dtype=dtype, num_blocks=blocks, max_batch_tokens=64, max_batch_seqs=seqs, prefill_chunk_size=32,
                     max_seq_len=160, cache_dtype=cache_dtype)
        outs.append(eng.generate(prompts, SamplingParams(max_tokens=20, temperature=0.0)))
        assert all(len(o) == 20 for o in outs[-1])
        stats = eng.stats()
        if blocks == 14:
            assert stats.preemptions > 0
        eng.close()
    # a request that starts again computes its decoded tokens as a portion: other sums, so an id may fall the other way now and then
    same = sum(a == b for x, y in zip(*outs) for a, b in zip(x, y))
    assert same >= 0.5 * 20 * len(prompts)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_other_plans(dtype):
    """Layers with a state beside layers with pages, a layer that reads another entry's keys through a window of its own, queries and keys
    without positions, a soft cap, and a mixer with a step of its own before the rotation."""
    import toy_kernels  # noqa: F401  (registers zk_toy_head_norm)
    from zse_amd.config import (AttentionSpec, BlockSpec, EmbeddingSpec, GatedMLPSpec, HeadSpec, LayerCall, ModelPlan, NormSpec, RotarySpec)
    from zse_amd.config.plan import NoPositionSpec
    from zse_amd.engine.loading import random_model
    from zse_amd.engine.runner import StepEntry, StepRunner
    from zse_amd.parts.attention import PagedAttention
    from zse_amd.parts.base import register_part, unregister_part
    from zse_amd.runtime.device import Runtime
    from toy_state import DecaySpec, toy_architecture
    from dataclasses import dataclass
    rt = Runtime.get()
    H, V, nh, nkv, hd = 64, 200, 4, 2, 48

    class UnitLengthAttention(PagedAttention):
        def between_product_and_rotation(self, ctx, qkv):
            s = self.spec
            ctx.rt.kernels(ctx.dtype).zk_toy_head_norm(qkv.ptr, qkv.shape[0], qkv.shape[1], s.num_heads + s.num_kv_heads, s.head_dim, ctx.stream)

    @dataclass(frozen=True)
    class UnitSpec(AttentionSpec):
        kind: str = "toy_unit_attention"

    def plan_of(cfg):
        norm = lambda n: NormSpec(H, 1e-6, False, n)
        names = lambda l, roles: {r: f"l{l}.attn.{r}" for r in roles}
        rotary = RotarySpec(hd, hd // 2, 1000.0)
        mixers = [AttentionSpec(H, nh, nkv, hd, 0.3, None, None, rotary, names(0, "qkvo")),
                  AttentionSpec(H, nh, nkv, hd, 0.3, 5.0, 20, rotary, names(1, "qo")),
                  DecaySpec(H, 0.75, "l2.mix.w"),
                  AttentionSpec(H, nh, 1, hd, 0.2, None, 24, NoPositionSpec(), names(3, "qkvo")),
                  UnitSpec(H, nh, nkv, 32, 2.0, None, None, RotarySpec(32, 32, 1000.0), names(4, "qkvo"))]
        layers = tuple(BlockSpec("prenorm", m, GatedMLPSpec(H, 96, "silu", {r: f"l{l}.ffn.{r}" for r in ("gate", "up", "down")}),
                                 {"pre_mixer": norm(f"l{l}.n1"), "pre_ffn": norm(f"l{l}.n2")}) for l, m in enumerate(mixers))
        return ModelPlan("ToyEightBitLM", H, V, 512, EmbeddingSpec(V, H, 1.0, "emb"), layers,
                         tuple(LayerCall(l, cache_of=0 if l == 1 else None) for l in range(5)), norm("final"), HeadSpec(V, H, None, "emb"))

    register_part("mixer", "toy_unit_attention", UnitLengthAttention)
    try:
        with toy_architecture("ToyEightBitLM", plan_of):
            model = random_model({"architectures": ["ToyEightBitLM"]}, dtype, seed=4, std=0.1, gain_std=0.1, rt=rt, std_of={"emb": 0.3})
            rng = np.random.default_rng(0)
            tokens, other = rng.integers(0, V, 70).tolist(), rng.integers(0, V, 90).tolist()

            def run(cache_dtype, cuts):
                runner = StepRunner(model, rt, dtype, page_size=16, cache_tokens=512, max_seqs=3, max_batch_tokens=128, max_model_len=256,
                                    cache_dtype=cache_dtype)
                rows, at = [], 0
                for i, n in enumerate(cuts):
                    z = runner.step([StepEntry("o", other[i:i + 1], []), StepEntry("r", tokens[at:at + n], list(range(n)))])
                    rows.append(z)
                    at += n
                runner.close()
                return np.concatenate(rows)

            plain = run(None, [70])
            for cache_dtype in FORMATS:
                whole, single, mixed = (run(cache_dtype, c) for c in ([70], [1] * 70, [30, 1, 1, 20, 18]))
                rounding = np.abs(whole - plain).max()
                # codes are a few hundredths of a value apart: the logits move, and by less than they are large
                assert 0 < rounding < 0.3 * np.abs(plain).max()
                for cut in (single, mixed):
                    err = np.abs(cut - whole)
                    if dtype == "float32":        # (as in the test of steps of every kind)
                        assert err.max() < rounding / 4 + F32_ATOL and np.median(err) < F32_ATOL, (cache_dtype, err.max(), rounding)
                    else:
                        assert err.max() < BF16_REL * np.abs(plain).max() + 2 * rounding, (cache_dtype, err.max(), rounding)
    finally:
        unregister_part("mixer", "toy_unit_attention")


def test_refused(tiny_folders):
    from zse_amd.engine.engine import Engine
    with pytest.raises(ValueError, match="16, 32"):
        Engine(tiny_folders[("A", "bfloat16")], block_size=4, num_blocks=8, cache_dtype="int8")
    with pytest.raises(ValueError, match="cache_dtype must be one of"):
        Engine(tiny_folders[("A", "bfloat16")], num_blocks=8, cache_dtype="int4")


def test_refused_by_a_mixer_that_does_not_serve_it():
    import dafotar_util as U
    from zse_amd.engine.loading import random_model
    from zse_amd.engine.runner import StepRunner
    from zse_amd.runtime.device import Runtime
    cfg = next(v for v in vars(U).values() if isinstance(v, dict) and v.get("architecture") == "Dafotar")
    model = random_model(cfg, "bfloat16", seed=0)
    with pytest.raises(ValueError, match="does not serve a cache in 8 bits"):
        StepRunner(model, Runtime.get(), "bfloat16", page_size=16, num_pages=8, max_seqs=2, max_model_len=64, cache_dtype="int8")


def test_bytes(tiny_folders):
    """Per token: codes of whole blocks of 64 channels and two scales, and one layer of each group in the compute type."""
    runner = make_runner(tiny_folders[("A", "bfloat16")], "bfloat16", page_size=16, num_pages=10, max_seqs=2, max_model_len=64, cache_dtype="fp8")
    layers, groups, nkv, hd = 2, 2, 2, 16
    assert runner.cache_bytes() == 11 * 16 * nkv * (layers * (2 * 64 + 8) + groups * 2 * hd * 2)
    assert runner.cache_token_bytes == layers * nkv * (2 * 64 + 8)
    runner.close()
    same = make_runner(tiny_folders[("A", "bfloat16")], "bfloat16", page_size=16, num_pages=10, max_seqs=2, max_model_len=64, cache_dtype="bf16")
    assert same.cache_dtype is None and all(c.format is None for c in same.caches)
    same.close()
