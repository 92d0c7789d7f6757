"""The Libulorn model - a gated attention with norms per head, a partial rotation and windows beside a linear one - with its cache in eight bits: on the
CPU through the plain kernel set, on the GPU through the kernels, against the plain model whose attention sees quantised keys and values."""
import os

import pytest
import torch

import plain_cache_quant as quant
import plain_libulorn as plain
import replay_modes
from helpers import assert_close, random_tokens
from libulorn_configs import LIB_A, _attention, _layer, _memory, _moe, _parallel
from test_cache_quant_engine import make_core

DEV = "cuda:0"
SIZES = {"small": (96, 4, 2, 32, 16), "wide": (128, 4, 2, 64, 32)}       # width, heads, key heads, numbers a head, rotated


def make_folder(tmp_path, size, dtype):
    from kvcache_b200.config import config_from_dict
    from kvcache_b200.weights import write_random_model
    width, heads, kv_heads, dim, rot = SIZES[size]
    side = lambda window, scaling: _attention(heads, kv_heads, dim, dim, 1.5 * dim ** -0.5, window, (10000.0, rot, scaling))
    data = {"architecture": "Libulorn", "vocab": 211, "width": width, "norm": {"eps": 1e-6}, "embedding": LIB_A["embedding"], "initializer_range": 0.08, "layers": [
        _layer(_parallel(side(37, (4.0, 1.0, 4.0, 32)), (3, 8, 16, 4.0, 6), 1.3, 0.7), _moe(4, 4, 24, 1.5, (40, 0.75))),     # all experts: no close calls
        _layer(_memory(2, 24, 16, 8.0), None),
        _layer(_parallel(side(None, None), (3, 8, 16, 4.0, 6), 1.2, 0.6), _moe(4, 4, 24, 1.5, (40, 0.75)))]}
    folder = os.path.join(str(tmp_path), "model")
    write_random_model(folder, config_from_dict(data), 3, dtype)
    return folder


def quantised_attention(store):
    def attention(h, w, p, m, eps):
        T, H, G, D = h.shape[0], int(m["heads"]), int(m["kv_heads"]), int(m["dim"])
        pos = torch.arange(T)
        q = plain.rotate(plain.unit(plain.linear(h, w[p + "q"]).view(T, H, D), eps) * w[p + "q.norm"], pos, m["rot"])
        k = plain.rotate(plain.unit(plain.linear(h, w[p + "k"]).view(T, G, D), eps) * w[p + "k.norm"], pos, m["rot"])
        v = plain.linear(h, w[p + "v"]).view(T, G, D)
        k, v = (quant.values(quant.to_pool(c, store), s).to(h.dtype) for c, s in (quant.quantise(x.double(), store) for x in (k, v)))
        seen = pos[None] <= pos[:, None]
        if m.get("mask"):
            seen &= pos[None] > pos[:, None] - int(m["mask"]["size"])
        s = torch.einsum("ihd,jhd->hij", q, k.repeat_interleave(H // G, 1)) * float(m["scale"])
        out = torch.einsum("hij,jhd->ihd", torch.softmax(s.masked_fill(~seen, float("-inf")), -1), v.repeat_interleave(H // G, 1))
        return plain.linear((out * torch.sigmoid(plain.linear(h, w[p + "g"]))[:, :, None]).reshape(T, H * D), w[p + "o"])
    return attention


def wanted(monkeypatch, folder, n, store):
    config, weights = plain.read_folder(folder)
    tokens = random_tokens(211, n, 7)
    exact = plain.logits_of(config, weights, tokens)
    monkeypatch.setattr(plain, "window_attention", quantised_attention(store))
    return config, weights, tokens, exact, plain.logits_of(config, weights, tokens)


def close(core, tokens, want, exact, sizes):
    """float32: as without quantisation (1e-4), and a few numbers beside a border of rounding that go the other way: each is one of thousands of
    roundings that together make the difference to the model without quantisation, of which a tenth is allowed."""
    rel = 1e-4 + 0.1 * float((want - exact).abs().max() / want.abs().max())
    assert_close(replay_modes.whole(core.runner, tokens), want, rel)
    assert_close(replay_modes.portions(core.runner, tokens, sizes), want, rel)
    assert_close(replay_modes.last_32_one_by_one(core.runner, tokens), want[-33:], rel)
    assert core.cache.used_pages() == 0


@pytest.mark.parametrize("store", quant.STORES)
def test_on_the_plain_kernel_set(tmp_path, monkeypatch, store):
    folder = make_folder(tmp_path, "small", torch.float32)
    _, _, tokens, exact, want = wanted(monkeypatch, folder, 75, store)
    core = make_core(folder, quant.QuantKernels(), "A", "float32", store, "cpu")
    assert all(g.spec.store == store for g in core.cache.groups) and len(core.cache.groups) == 2
    close(core, tokens, want, exact, [2, 17, 3, 31, 1, 1, 20])


@pytest.mark.gpu
@pytest.mark.parametrize("store", quant.STORES)
@pytest.mark.parametrize("size", SIZES)
def test_in_float32(tmp_path, monkeypatch, size, store):
    from kvcache_b200.kernels.api import CudaKernels
    folder = make_folder(tmp_path, size, torch.float32)
    _, _, tokens, exact, want = wanted(monkeypatch, folder, 210, store)
    core = make_core(folder, CudaKernels(DEV), "A", "float32", store, DEV, page_size=16)
    close(core, tokens, want, exact, [2, 140, 3, 31, 1, 1, 32])
    core.kernels.check_errors()


def as_rounding_alone(got, want, spread):
    """Errors as a distribution, against what rounding every product to bfloat16 does to the plain model that quantises (`spread`).  That is more than the 2 %
    of the largest logit which hold a model without quantisation: a number that is off by 2^-9 of itself goes to another code one time in sixteen (a step of e4m3
    is 2^-4 of its number, and 2^-8 on either side of a border are 2^-4 of a step), and then by a whole step - by a quarter of what quantising makes of all
    numbers, root mean square.  The plain model's own median is 2.0 to 3.4 % for these four.  So the median is held to 1.5 times the plain model's, the k-th
    largest to 4 times the plain model's k-th largest (at least 1 % of the largest logit) but for the largest 2 %, and none to twice its largest."""
    err, scale = (got.detach().double().cpu() - want).abs().max(dim=1).values, float(want.abs().max())
    assert torch.isfinite(err).all() and float(err.max()) <= 2 * float(spread.max())
    e, sp = torch.sort(err, descending=True).values, torch.sort(spread, descending=True).values
    over = e > 4 * torch.clamp(sp[torch.arange(len(e)) * len(sp) // len(e)], min=0.01 * scale)
    assert not over[max(1, len(e) // 50):].any()
    assert float(err.median()) <= 1.5 * float(spread.median())


@pytest.mark.gpu
@pytest.mark.parametrize("store", quant.STORES)
@pytest.mark.parametrize("size", SIZES)
def test_in_bfloat16(tmp_path, monkeypatch, size, store):
    from kvcache_b200.kernels.api import CudaKernels
    folder = make_folder(tmp_path, size, torch.bfloat16)
    config, weights, tokens, _, want = wanted(monkeypatch, folder, 210, store)
    with plain.rounding(torch.bfloat16):
        spread = (plain.logits_of(config, weights, tokens) - want).abs().max(dim=1).values
    kernels = CudaKernels(DEV)
    core = make_core(folder, kernels, "A", "bfloat16", store, DEV, page_size=16)
    as_rounding_alone(replay_modes.whole(core.runner, tokens), want, spread)
    as_rounding_alone(replay_modes.portions(core.runner, tokens, [2, 140, 3, 31, 1, 1, 32]), want, spread)
    as_rounding_alone(replay_modes.last_32_one_by_one(core.runner, tokens), want[-33:], spread[-33:])
    kernels.check_errors()
    assert kernels.launch_counts["append_quant"] and kernels.launch_counts["attention_quant"] and kernels.launch_counts["cache_expand"]
