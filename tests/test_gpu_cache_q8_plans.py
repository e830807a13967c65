"""A cache in 8 bits under other plans and through the engine, against runs in float64 that round keys and values likewise."""
from dataclasses import dataclass

import numpy as np
import pytest

from conftest import TINY
from gpu_util import BF16_REL, F32_ATOL
from plain import gemma2_plain as P
from test_gpu_cache_q8_engine import FORMATS, held, reference

pytestmark = pytest.mark.gpu

F64 = np.float64


def off_by(dtype, want, rounding):
    """What logits may be off by, where ``rounding`` is what the rounding of all keys and values changes (the reasons: the test of steps
    of every kind): in 32 bits a value moved across a code's border now and then, in 16 what 16 bits are off by and twice the rounding."""
    return rounding / 4 + F32_ATOL if dtype == "float32" else BF16_REL * np.abs(want).max() + 2 * rounding


H, V, NH, NKV, HD = 64, 200, 4, 2, 48


def unit(x):
    return x / np.sqrt((x * x).sum(-1, keepdims=True) + 1e-12)


def turned(x, rotary, theta):
    """The first ``rotary`` channels of every head in pairs (i, i + rotary / 2), the others as they are."""
    return np.concatenate([P.rope(x[..., :rotary], np.arange(len(x)), theta, F64), x[..., rotary:]], axis=-1) if rotary else x


def plain(w, tokens, form):
    """[T, V] logits of the plan below; ``form``: what keys and values are held as (None: as they are)."""
    T, pos = len(tokens), np.arange(len(tokens))
    keep = (lambda x: x) if form is None else (lambda x: held(x, form))
    mm = lambda x, name: x @ w[name].astype(F64).T
    h = w["emb"][np.asarray(tokens)].astype(F64)
    # key heads, channels, turned channels, scale, cap, window, whose keys
    specs = [(NKV, HD, HD // 2, 0.3, None, None, 0), (NKV, HD, HD // 2, 0.3, 5.0, 20, 0), None, (1, HD, 0, 0.2, None, 24, 3), (NKV, 32, 32, 2.0, None, None, 4)]
    stored = {}
    for l, s in enumerate(specs):
        x = P.rmsnorm(h, w[f"l{l}.n1"], 1e-6, F64, unit_offset=False)
        if s is None:
            state, rows = np.zeros(H), []
            for row in x:
                state = 0.75 * state + row
                rows.append(state)
            h = h + mm(np.stack(rows), "l2.mix.w")
        else:
            nkv, hd, rotary, scale, cap, window, of = s
            norm = unit if l == 4 else (lambda a: a)
            q = turned(norm(mm(x, f"l{l}.attn.q").reshape(T, NH, hd)), rotary, 1000.0)
            if of == l:
                k = turned(norm(mm(x, f"l{l}.attn.k").reshape(T, nkv, hd)), rotary, 1000.0)
                stored[l] = keep(k), keep(mm(x, f"l{l}.attn.v").reshape(T, nkv, hd))
            o = P.attention(q, *stored[of], pos, scale, cap, window, F64)
            h = h + mm(o.reshape(T, -1), f"l{l}.attn.o")
        x = P.rmsnorm(h, w[f"l{l}.n2"], 1e-6, F64, unit_offset=False)
        g = mm(x, f"l{l}.ffn.gate")
        h = h + mm(g / (1 + np.exp(-g)) * mm(x, f"l{l}.ffn.up"), f"l{l}.ffn.down")
    return mm(P.rmsnorm(h, w["final"], 1e-6, F64, unit_offset=False), "emb")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_layers_of_every_kind(tmp_path, dtype):
    """Layers with a state beside layers with pages, a layer that reads another entry's keys through a window and a cap of its own, a part of
    the head turned, no positions, a mixer with a step of its own before the rotation: portions, single tokens and both."""
    import toy_kernels  # noqa: F401  (registers zk_toy_head_norm)
    from zse_amd.config import (AttentionSpec, BlockSpec, EmbeddingSpec, GatedMLPSpec, HeadSpec, LayerCall, ModelPlan, NormSpec, RotarySpec)
    from zse_amd.config.plan import NoPositionSpec
    from zse_amd.engine.loading import load_model
    from zse_amd.engine.runner import StepEntry, StepRunner
    from zse_amd.parts.attention import PagedAttention
    from zse_amd.parts.base import register_part, unregister_part
    from zse_amd.runtime.device import Runtime
    from zse_amd.weights import write_random_model
    from zse_amd.weights.safetensors import read_folder_f32
    from toy_state import DecaySpec, toy_architecture
    rt = Runtime.get()

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
        rotary = RotarySpec(HD, HD // 2, 1000.0)
        mixers = [AttentionSpec(H, NH, NKV, HD, 0.3, None, None, rotary, names(0, "qkvo")),
                  AttentionSpec(H, NH, NKV, HD, 0.3, 5.0, 20, rotary, names(1, "qo")),
                  DecaySpec(H, 0.75, "l2.mix.w"),
                  AttentionSpec(H, NH, 1, HD, 0.2, None, 24, NoPositionSpec(), names(3, "qkvo")),
                  UnitSpec(H, NH, NKV, 32, 2.0, None, None, RotarySpec(32, 32, 1000.0), names(4, "qkvo"))]
        layers = tuple(BlockSpec("prenorm", m, GatedMLPSpec(H, 96, "silu", {r: f"l{l}.ffn.{r}" for r in ("gate", "up", "down")}),
                                 {"pre_mixer": norm(f"l{l}.n1"), "pre_ffn": norm(f"l{l}.n2")}) for l, m in enumerate(mixers))
        return ModelPlan("ToyHeldLM", H, V, 512, EmbeddingSpec(V, H, 1.0, "emb"), layers,
                         tuple(LayerCall(l, cache_of=0 if l == 1 else None) for l in range(5)), norm("final"), HeadSpec(V, H, None, "emb"))

    register_part("mixer", "toy_unit_attention", UnitLengthAttention)
    try:
        with toy_architecture("ToyHeldLM", plan_of):
            folder = write_random_model(str(tmp_path / "m"), {"architectures": ["ToyHeldLM"]}, seed=4, std=0.1, gain_std=0.1, dtype=dtype,
                                        std_of={"emb": 0.3})
            w, model = read_folder_f32(folder), load_model(folder, dtype, rt)
            rng = np.random.default_rng(0)
            tokens, other = rng.integers(0, V, 70).tolist(), rng.integers(0, V, 90).tolist()
            exact = plain(w, tokens, None)
            for cache_dtype, form in FORMATS.items():
                want = plain(w, tokens, form)
                rounding = np.abs(want - exact).max()
                assert rounding > 0
                for cuts in ([70], [1] * 70, [30, 1, 1, 20, 18]):
                    runner = StepRunner(model, rt, dtype, page_size=16, cache_tokens=512, max_seqs=3, max_batch_tokens=128, max_model_len=256,
                                        cache_dtype=cache_dtype)
                    rows, at = [], 0
                    for i, n in enumerate(cuts):
                        rows.append(runner.step([StepEntry("o", other[i:i + 1], []), StepEntry("r", tokens[at:at + n], list(range(n)))]))
                        at += n
                    runner.close()
                    err = np.abs(np.concatenate(rows) - want)
                    assert err.max() < off_by(dtype, want, rounding), (cache_dtype, len(cuts), err.max(), rounding, np.abs(want).max())
                    assert dtype != "float32" or np.median(err) < F32_ATOL, (cache_dtype, len(cuts), np.median(err))
    finally:
        unregister_part("mixer", "toy_unit_attention")


@pytest.mark.parametrize("cache_dtype", ["int8", "float8_e4m3"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_every_generated_id_is_one_of_the_largest(monkeypatch, tiny_folders, dtype, cache_dtype):
    """Through the engine, in portions beside decoded tokens, with room for everybody and with requests that give their pages up and start
    again: each id's logit, after all that came before it, is the largest but for what logits may be off by."""
    from zse_amd.engine.engine import Engine
    from zse_amd.sampling import SamplingParams
    folder = tiny_folders[("A", dtype)]
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, 512, n).tolist() for n in (5, 70, 33, 16, 1, 100)]
    for blocks in (64, 14):
        eng = Engine(folder, dtype=dtype, num_blocks=blocks, max_batch_tokens=64, max_batch_seqs=6, prefill_chunk_size=32, max_seq_len=160,
                     cache_dtype=cache_dtype)
        outs = eng.generate(prompts, SamplingParams(max_tokens=20, temperature=0.0))
        assert (eng.stats().preemptions > 0) == (blocks == 14)
        eng.close()
        for p, out in zip(prompts, outs):
            assert len(out) == 20
            z = reference(monkeypatch, "A", dtype, folder, p + out[:-1], FORMATS[cache_dtype])
            rounding = np.abs(z - reference(monkeypatch, "A", dtype, folder, p + out[:-1], None)).max()
            z = z[len(p) - 1:]
            short = z.max(axis=1) - z[np.arange(20), out]
            assert (short <= 2 * off_by(dtype, z, rounding)).all(), (blocks, len(p), short.max(), rounding)
            assert np.median(short) == 0


@pytest.mark.parametrize("cache_dtype", ["int8", "float8_e4m3"])
def test_company_leaves_a_requests_bits_in_32_bits(tiny_folders, cache_dtype):
    """Cut alike, alone and beside others that come, decode and end."""
    from gpu_util import make_runner
    from zse_amd.engine.runner import StepEntry
    rng = np.random.default_rng(1)
    tokens = rng.integers(0, 512, 90).tolist()
    cuts = [30, 1, 1, 20, 1, 1, 1, 12] + [1] * 10
    got = []
    for company in (False, True):
        runner = make_runner(tiny_folders[("A", "float32")], "float32", page_size=16, num_pages=60, max_seqs=6, max_batch_tokens=256, max_model_len=256,
                             use_graphs=True, cache_dtype=cache_dtype)
        rows, at = [], 0
        for i, n in enumerate(cuts):
            entries = [StepEntry("r", tokens[at:at + n], list(range(n)))]
            at += n
            if company:
                if i == 9:
                    runner.finish("x")
                entries = ([StepEntry("x", tokens[:40] if i == 0 else [i], [0])] if i < 9 else []) + entries
                entries += [StepEntry(j, [7 + i, j, 3][:1 + (i + j) % 3], []) for j in range(min(i, 4))]
            z = runner.step(entries)
            first = 1 if company and i < 9 else 0
            rows.append(z[first:first + n])
        runner.close()
        got.append(np.concatenate(rows))
    assert np.array_equal(*got)
