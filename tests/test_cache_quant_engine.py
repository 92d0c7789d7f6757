"""The engine with its cache in eight bits: host logic on the CPU through the plain kernel set, the kernels on the GPU, both against a plain model
whose layers attend to quantised keys and values."""
import json

import pytest
import torch

import plain_cache_quant as plain
import replay_modes
from helpers import assert_close, random_tokens
from plain_qwen2 import logits_of, read_folder
from tiny_configs import PAGE_SIZE, make_model_folder

DEV = "cuda:0"
# float32: the codes are the plain model's but where a number lies within float32's rounding of a border; one such code moves one number of one
# key or value by a step of at most 2^-3 of itself.
REL32 = 2e-3


def make_core(folder, kernels, name, dtype, store, device, **options):
    from kvcache_b200.config.options import EngineOptions
    from kvcache_b200.engine.core import EngineCore
    fields = dict(dtype=dtype, cache_dtype=store, page_size=PAGE_SIZE[name], num_pages=64, max_running=4, max_tokens_per_step=512, max_model_len=512,
                  use_graphs=False, device=device)
    return EngineCore(folder, EngineOptions(**{**fields, **options}), kernels=kernels)


@pytest.mark.parametrize("store", plain.STORES)
@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_engine_on_the_plain_kernel_set(tmp_path, name, store):
    folder = make_model_folder(tmp_path, name)
    core = make_core(folder, plain.QuantKernels(), name, "float32", store, "cpu")
    config, weights = read_folder(folder)
    tokens = random_tokens(config["vocab_size"], 75, 1)
    want = plain.logits_of(config, weights, tokens, store)
    got = replay_modes.whole(core.runner, tokens)
    assert_close(got, want, REL32)
    assert_close(replay_modes.portions(core.runner, tokens, [2, 17, 3, 31, 1, 1, 20]), want, REL32)
    assert_close(replay_modes.last_32_one_by_one(core.runner, tokens), want[-33:], REL32)
    assert core.cache.used_pages() == 0
    # The quantisation is there: the plain model without it is further from the engine than the one with it.
    exact = logits_of(config, weights, tokens)
    assert (got.double().cpu() - exact).abs().max() > 2 * (got.double().cpu() - want).abs().max()


@pytest.mark.parametrize("store", plain.STORES)
def test_what_the_cache_holds(tmp_path, store):
    folder = make_model_folder(tmp_path, "C")                # two groups: full and windowed layers
    core = make_core(folder, plain.QuantKernels(), "C", "float32", store, "cpu")
    D, Hkv, layers = 48, 2, 4
    assert core.cache.kv_bytes_per_token() == layers * Hkv * 2 * (D + 1)
    for group in core.cache.groups:
        assert group.spec.store == store and group.k_pool.dtype == plain.STORE_DTYPES[store] and group.k_scales.shape == group.k_pool.shape[:-1]
    view = core.cache.step_view([torch.zeros(1, 1, dtype=torch.int32)] * 2).kv_view(0, True)
    assert view.k_scales.data_ptr() == core.cache.groups[0].k_scales[0].data_ptr() and view.v_scales is not None
    plain_core = make_core(folder, plain.QuantKernels(), "C", "float32", "auto", "cpu")
    assert all(g.spec.store is None and g.k_scales is None for g in plain_core.cache.groups)


def test_options_that_are_refused(tmp_path):
    from kvcache_b200.config.options import EngineOptions
    with pytest.raises(ValueError, match="cache_dtype"):
        EngineOptions(num_pages=4, cache_dtype="fp4")


def _mixer(**changes):
    from kvcache_b200.parts.attention import GQAAttention
    fields = dict(qkv_bias=False, out_bias=False, position=None, window=None, prefix="p.", dtype="bfloat16")
    return GQAAttention(64, 4, 2, 32, **{**fields, **changes})


@pytest.mark.parametrize("changes, words", [
    (dict(value_dim=16), "another size"), (dict(qk_norm_eps=1e-6, qk_norm_scope="all"), "whole projections"),
    (dict(qk_norm_eps=1e-6, qk_norm_after_rotation=True), "after the rotation"), (dict(value_mix="source"), "blended"),
    (dict(q_temperature=(0.1, 8)), "temperature")])
def test_layers_that_are_refused(changes, words):
    with pytest.raises(ValueError, match=words):
        _mixer(**changes).store_cache("e4m3")


def test_layers_that_are_taken():
    for changes in (dict(), dict(window=64, keep_first=3, sink=1.0), dict(chunk=16), dict(qk_norm_eps=1e-6), dict(score_cap=5.0, distance_bias="geometric"),
                    dict(own_kv=False), dict(head_gate="g.weight")):
        mixer = _mixer(**changes)
        mixer.store_cache("int8")
        assert mixer.cache_store == "int8" and (mixer.cache_spec() is None or mixer.cache_spec().store == "int8")
    with pytest.raises(ValueError, match="held as one of"):
        _mixer().store_cache("fp4")


def test_heads_that_no_kernel_takes_in_eight_bits():
    from kvcache_b200.parts.attention import GQAAttention
    wide = GQAAttention(64, 4, 2, 1040, qkv_bias=False, out_bias=False, position=None, window=None, prefix="p.", dtype="bfloat16")
    with pytest.raises(ValueError, match="1,024"):
        wide.store_cache("int8")


def test_a_model_with_pages_that_cannot_be_held_so(tmp_path):
    from kakipel_configs import CONFIGS
    from kvcache_b200.config import config_from_dict
    from kvcache_b200.weights import write_random_model
    folder = str(tmp_path / "latent")
    config = config_from_dict(next(iter(CONFIGS.values())))
    write_random_model(folder, config, 0, torch.float32)
    with pytest.raises(ValueError, match="layer 0: LatentAttention keeps its pages"):
        make_core(folder, plain.QuantKernels(), "A", "float32", "e4m3", "cpu", max_model_len=None)


# ---- on the GPU --------------------------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def kernels():
    from kvcache_b200.kernels.api import CudaKernels
    return CudaKernels(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("store", plain.STORES)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
def test_engine_on_the_gpu(tmp_path, kernels, name, dtype, store):
    folder = make_model_folder(tmp_path, name, dtype=torch.bfloat16)
    config, weights = read_folder(folder)
    tokens = random_tokens(config["vocab_size"], 410, 5)
    want = plain.logits_of(config, weights, tokens, store)
    exact = logits_of(config, weights, tokens)
    scale = want.abs().max().item()
    # bfloat16: 3e-2 of the largest logit as without quantisation; activations that are off by 2^-8 send some numbers to a neighbouring code,
    # which makes no more noise than the quantisation itself: what that does to a logit at worst is allowed twice.
    rel = REL32 if dtype == "float32" else 3e-2 + 2 * (want - exact).abs().max().item() / scale
    core = make_core(folder, kernels, name, dtype, store, DEV)
    assert_close(replay_modes.whole(core.runner, tokens), want, rel)
    assert_close(replay_modes.portions(core.runner, tokens, [2, 170, 3, 31, 1, 1, 202]), want, rel)
    assert_close(replay_modes.last_32_one_by_one(core.runner, tokens), want[-33:], rel)
    kernels.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["B", "D"])
def test_mixed_batches_with_reused_pages(tmp_path, kernels, name):
    folder = make_model_folder(tmp_path, name, dtype=torch.bfloat16)
    config, weights = read_folder(folder)
    core = make_core(folder, kernels, name, "float32", "int8", DEV, num_pages=replay_modes.mixed_pool_tokens() // PAGE_SIZE[name])
    seqs = {k: random_tokens(config["vocab_size"], n, 10 + i) for i, (k, n) in enumerate(replay_modes.MIXED_LENGTHS)}
    got = replay_modes.mixed(core.runner, seqs)
    for k, tokens in seqs.items():
        assert_close(got[k], plain.logits_of(config, weights, tokens, "int8"), REL32, k)
    kernels.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("store", plain.STORES)
def test_generation_is_the_same_with_and_without_graphs(tmp_path, kernels, store):
    from kvcache_b200 import LLM, SamplingParams
    folder = make_model_folder(tmp_path, "D", dtype=torch.bfloat16)
    prompts = [random_tokens(270, n, 20 + n) for n in (5, 140, 33)]
    params = SamplingParams(max_new_tokens=24, temperature=0.0, ignore_eos=True)
    out = []
    for graphs in (True, False):
        llm = LLM(folder, dtype="bfloat16", cache_dtype=store, page_size=16, num_pages=64, max_running=4, max_tokens_per_step=256, use_graphs=graphs)
        llm.core.runner.split_mixed_steps = False            # a mixed step cut in parts rounds otherwise
        out.append(llm.generate(prompts, params))
        assert all(len(o) == 24 for o in out[-1])
    assert out[0] == out[1]
    assert llm.core.kernels.launch_counts["append_quant"] and llm.core.kernels.launch_counts["attention_quant"]


@pytest.mark.gpu
def test_command_lines(tmp_path):
    import subprocess
    import sys
    folder = make_model_folder(tmp_path, "D", dtype=torch.bfloat16)
    run = lambda module, *args, text: subprocess.run([sys.executable, "-m", f"kvcache_b200.cli.{module}", *args], input=text, capture_output=True, text=True,
                                                     check=True, timeout=300).stdout
    one = run("infer", folder, "6", "--cache-dtype", "int8", text="1 2 3").split()
    many = run("serve", folder, "--cache-dtype", "int8", "--ignore-eos", text="2\n6 1 2 3\n4 7 8\n").splitlines()
    assert len(one) == 6 and many[0].split() == one and len(many[1].split()) == 4
    line = json.dumps({"step": 0, "entries": [{"id": "a", "tokens": [1, 2, 3], "want": [2]}], "end": ["a"]})
    assert "done 0" in run("trace", "--model", folder, "--dtype", "float32", "--cache-dtype", "e4m3", "--out", str(tmp_path / "out"), "--max-tokens", "64", text=line + "\n")
    assert (tmp_path / "out" / "0.f32").stat().st_size == 270 * 4
