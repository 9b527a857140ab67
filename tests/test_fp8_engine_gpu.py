"""The engine with keys and values in 8 bits, against the plain models whose attention sees quantised keys and values."""
import os
import subprocess
import sys

import pytest
import torch

import plain_fp8_cache as fp8
import plain_qwen2moe as plain
import plain_safepel as safepel
import safepel_configs
from tiny_configs import CONFIGS, make_folder

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def quantised(x):
    """[tokens, heads, dim] as the cache holds it."""
    return fp8.values(*fp8.quantise(x)).to(x.dtype)


@pytest.fixture
def plain_in_8_bits(monkeypatch):
    own = plain.attention
    monkeypatch.setattr(plain, "attention", lambda q, k, v, window: own(q, quantised(k), quantised(v), window))
    return own


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("fp8")
    return {name: make_folder(tmp, name, std=0.2) for name in CONFIGS}


def engine(folder, dtype="float32", **kw):
    from ferrox_b200 import Engine

    kw = {**dict(page_size=16, n_pages=48, max_slots=4, kv_cache="fp8"), **kw}
    return Engine.from_folder(folder, dtype=dtype, **kw)


def logits_of(eng, prompt, cuts):
    """Logits of every position of ``prompt`` run in portions of the given sizes (the last repeats)."""
    from ferrox_b200 import StepEntry

    slot, out, at, i = eng.open_request(), [], 0, 0
    while at < len(prompt):
        n = min(cuts[min(i, len(cuts) - 1)], len(prompt) - at)
        out.append(eng.step([StepEntry(slot, prompt[at:at + n], want=list(range(n)))]).cpu().clone())
        at, i = at + n, i + 1
    eng.close_request(slot)
    return torch.cat(out)


PROMPT = [(7 * i * i + 3 * i + 11) % 200 for i in range(90)]


@pytest.mark.parametrize("name", list(CONFIGS))
@pytest.mark.parametrize("cuts", [[90], [1], [40, 30, 7, 1]])
def test_logits_in_32_bits(folders, plain_in_8_bits, name, cuts):
    """Both sides quantise rows that differ in their last bits: an element next to the middle between two e4m3 numbers may fall to
    either side on them, one element of a position by a step (2^-3 of it at most).  So the median is held to 32-bit rounding
    through the model (the bound of the tests without a quantised cache, 2e-5, times 5 for the median over fewer exact
    positions) and every position to what such a step may do."""
    cfg, w = plain.load_model(folders[name])
    want = plain.forward(cfg, w, PROMPT)
    got = logits_of(engine(folders[name]), PROMPT, cuts)
    off = (got - want).abs().amax(1) / want.abs().max()
    assert off.median() < 1e-4 and off.max() < 5e-2
    # the test can tell: without the quantisation the plain logits are somewhere else
    plain.attention = plain_in_8_bits
    assert ((plain.forward(cfg, w, PROMPT) - got).abs().amax(1) / want.abs().max()).median() > 1e-3


@pytest.mark.parametrize("name", list(CONFIGS))
def test_greedy_generation(folders, plain_in_8_bits, name):
    cfg, w = plain.load_model(folders[name])
    prompts = [[5, 9, 200, 31], [7], list(range(40, 75))]
    want = [plain.greedy(cfg, w, p, 12) for p in prompts]
    eng = engine(folders[name])
    assert eng.generate(prompts, max_new_tokens=12) == want
    assert eng.generate(prompts, max_new_tokens=12, max_batch_tokens=5) == want
    eng.cache.check_invariants()
    assert eng.cache.n_free_slots == 4


@pytest.mark.parametrize("name", list(CONFIGS))
def test_replayed_steps_give_what_eager_ones_give(folders, name):
    prompts = [[5, 9, 200, 31], [7, 8], list(range(40, 75))]
    outs = [engine(folders[name], dtype="bfloat16", cuda_graphs=g).generate(prompts, max_new_tokens=40) for g in (True, False)]
    assert outs[0] == outs[1] and all(len(o) == 40 for o in outs[0])


def test_half_the_bytes(folders):
    a, b = (engine(folders["A"], dtype="bfloat16", kv_cache=kv) for kv in (None, "fp8"))
    G, D = 2, 16
    assert b.cache.kv_bytes() * 2 * D == a.cache.kv_bytes() * (D + 1)
    assert a.cache.layer_cache(0).fp8 is False and b.cache.layer_cache(0).fp8 is True
    assert b.cache.layer_cache(0).k.dtype == torch.float8_e4m3fn and b.cache.layer_cache(0).pages["k_exp"].shape == (48, G, 16)


def test_preempted_requests_come_back_the_same(folders, plain_in_8_bits):
    cfg, w = plain.load_model(folders["A"])
    prompts = [[i + 1, i + 3, i + 7, 99, 4, 8, 15, 16] for i in range(4)]
    want = [plain.greedy(cfg, w, p, 20) for p in prompts]
    outs, stats = engine(folders["A"], page_size=4, n_pages=14).generate(prompts, max_new_tokens=20, return_stats=True)
    assert stats["preemptions"] >= 1 and outs == want


@pytest.mark.parametrize("name", ["A", "B", "C", "E"])
@pytest.mark.parametrize("cuts", [[90], [1]])
def test_windowed_capped_attention_beside_another_mixer(tmp_path, monkeypatch, name, cuts):
    """Safepel: a window, capped scores, rotation in adjacent pairs, values that are the keys before it, beside a recurrence."""
    from ferrox_b200 import Engine

    folder = safepel_configs.make_folder(tmp_path, name)
    cfg, w = plain.load_model(folder)
    prompt = [t % cfg["vocab"] for t in PROMPT]

    def attention(h, w, p, m, positions):
        T, H, G, D = h.shape[0], m["heads"], m["kv_heads"], m["dim"]
        q = safepel.rotate_adjacent((h @ w[p + "q"].T).view(T, H, D), positions, m["rot"]["base"], m["rot"]["dims"])
        k = (h @ w[p + "k"].T).view(T, G, D)
        kr, v = quantised(safepel.rotate_adjacent(k, positions, m["rot"]["base"], m["rot"]["dims"])), quantised(k)
        far = positions[:, None] - positions[None, :]
        out = h.new_zeros(T, H, D)
        for hd in range(H):
            s = m["softcap"] * torch.tanh((q[:, hd] @ kr[:, hd // (H // G)].T) * m["scale"] / m["softcap"])
            out[:, hd] = torch.softmax(s.masked_fill((far < 0) | (far >= m["mask"]["size"]), float("-inf")), -1) @ v[:, hd // (H // G)]
        return out.reshape(T, H * D) @ w[p + "o"].T

    monkeypatch.setattr(safepel, "capped_window_attention", attention)
    want = safepel.forward(cfg, w, prompt)
    got = logits_of(Engine.from_folder(folder, dtype="float32", page_size=16, n_pages=48, max_slots=4, kv_cache="fp8"), prompt, cuts)
    off = (got - want).abs().amax(1) / want.abs().max()
    assert off.median() < 1e-4 and off.max() < 5e-2


@pytest.mark.parametrize("name", ["A", "B", "C", "E"])
def test_portions_beside_another_mixer(tmp_path, monkeypatch, name):
    """Portions of so few tokens that the mixers of a sum run side by side, prompts by the tiled kernels and by the decode kernel."""
    test_windowed_capped_attention_beside_another_mixer(tmp_path, monkeypatch, name, [20, 33, 9, 8, 12])


def test_models_with_other_caches_are_refused(tmp_path):
    import bobepel_configs
    from ferrox_b200 import Engine

    with pytest.raises(ValueError, match="not held in 8 bits"):
        Engine.from_random(bobepel_configs.BOBEPEL_A, kv_cache="fp8")
    with pytest.raises(ValueError, match="kv_cache='int8'"):
        Engine.from_random(CONFIGS["A"][0], kv_cache="int8")


def test_command_line(folders):
    cmd = [sys.executable, "-m", "ferrox_b200", "-m", folders["A"], "--tokens", "5,9,200,31", "-n", "8", "--temp", "0", "--repeat-penalty", "1",
           "--dtype", "float32", "--page-size", "16", "--num-pages", "16"]
    outs = []
    for kv in ("model", "fp8"):
        r = subprocess.run(cmd + ["--kv-cache", kv], cwd=ROOT, capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr
        outs.append([int(t) for t in r.stdout.split()])
    assert outs[1] == engine(folders["A"]).generate([5, 9, 200, 31], max_new_tokens=8) and len(outs[0]) == 8
