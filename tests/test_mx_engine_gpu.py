"""Models served with matrices in 4 bits (weights="mxfp4") and rows in 8 (rows="mxfp8"), against the plain implementations with the same rounding."""

import subprocess
import sys

import numpy as np
import pytest
import torch

import plain_gpt2 as plain
import plain_lafanex
import plain_larulorn
import plain_mx
import trace_tools as tt
from conftest import CONFIG_A, TOL

pytestmark = pytest.mark.gpu

# what is rounded: the plan's spec kinds and the tensors that they read through products alone
IN_4_BITS = {"attention": ("qkv_weight", "out_weight"), "dense_ffn": ("up_weight", "down_weight"), "scored_attention": ("q", "k", "v", "gate", "out"),
             "clamped_glu": ("gate", "up", "down"), "gated_ffn": ("gate", "up", "down"), "selective_scan": ("in", "out")}


def rounded(tensors, plan, prefixes=("",), through_bf16=False):
    """The tensors with the plan's matrices in 4 bits, along their input features (rounded to bfloat16 first on that path)."""
    out = dict(tensors)
    count = 0
    for layer in plan.layers:
        for spec in (layer.mixer, layer.ffn):
            for key in IN_4_BITS.get(getattr(spec, "kind", ""), ()):
                src = spec.tensors.get(key)
                if src is None:
                    continue
                name = next(p + src.name for p in prefixes if p + src.name in tensors)
                w = tensors[name] if not through_bf16 else plain.round_to_bf16(tensors[name])
                w = w.T if src.layout == "in_out" else w
                q = plain_mx.values(*plain_mx.quantize(w, plain_mx.E2M1, 2), plain_mx.E2M1)
                out[name] = q.T if src.layout == "in_out" else q
                count += 1
    assert count
    return out


def core_of(model_dir, steps, dtype="bfloat16", **kw):
    from liyab_amd.engine import EngineCore

    return EngineCore(model_dir, dtype=dtype, page_size=16, max_tokens=tt.max_live_tokens(steps), max_requests=8, **kw)


def plan_of(config):
    from liyab_amd.config.registry import config_from_dict

    return config_from_dict(config).plan()


SCHEDULES = {"whole": tt.schedule_whole, "portions": tt.schedule_portions, "mixed": lambda reqs: tt.schedule_mixed(reqs, seed=3, decode_tail=9)}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_gpt2_in_4_bits(model_dirs, plain_models, name, dtype):
    """Logits of the plain implementation over the rounded matrices, within the tolerances of the unrounded model's tests, however the work is cut."""
    config, tensors = plain_models[name]
    plan = plan_of(config)
    mine = rounded(tensors, plan, through_bf16=dtype == "bfloat16")
    if dtype == "bfloat16":
        mine = {k: (plain.round_to_bf16(v) if v.ndim >= 2 and ("wte" in k or "wpe" in k) else v) for k, v in mine.items()}
    V = config["vocab_size"]
    reqs = {f"r{i}": tt.random_tokens(40 + i, n, V) for i, n in enumerate([70, 21, 1, 100])}
    ref = {rid: plain.forward(config, mine, toks) for rid, toks in reqs.items()}
    for label, make in SCHEDULES.items():
        steps = make(reqs)
        core = core_of(model_dirs[name], steps, dtype, weights="mxfp4")
        got = tt.run_schedule(core, steps)
        tt.check_against_plain(got, reqs, ref, TOL[dtype], f"mxfp4 {name} {dtype} {label}", family=f"GPT-2 in 4 bits, {dtype}")
        del core


def rows8(x):
    return plain_mx.values(*plain_mx.quantize(x, plain_mx.E4M3, 8), plain_mx.E4M3)


def forward_rows8(config, tensors, ids):
    """plain_gpt2.forward with every product's rows rounded to 8 bits."""
    x = plain.embed(tensors["wte.weight"], tensors["wpe.weight"], ids, range(len(ids)))
    eps = config.get("layer_norm_epsilon", 1e-5)
    act = plain.ACTIVATIONS[config.get("activation_function", "gelu_new")]
    for layer in range(config["n_layer"]):
        p = f"h.{layer}"
        h = rows8(plain.layer_norm(x, tensors[p + ".ln_1.weight"], tensors[p + ".ln_1.bias"], eps))
        q, k, v = (plain.round_to_bf16(t) for t in plain.qkv_projection(h, tensors[p + ".attn.c_attn.weight"], tensors[p + ".attn.c_attn.bias"]))
        att = plain.round_to_bf16(plain.causal_attention(q, k, v, config["n_head"], plain.attention_scale(config, layer)))
        x = x + rows8(att) @ tensors[p + ".attn.c_proj.weight"] + tensors[p + ".attn.c_proj.bias"]
        h = rows8(plain.layer_norm(x, tensors[p + ".ln_2.weight"], tensors[p + ".ln_2.bias"], eps))
        inner = plain.round_to_bf16(act(h @ tensors[p + ".mlp.c_fc.weight"] + tensors[p + ".mlp.c_fc.bias"]))
        x = x + rows8(inner) @ tensors[p + ".mlp.c_proj.weight"] + tensors[p + ".mlp.c_proj.bias"]
    return plain.lm_head(x, tensors, config)


@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_gpt2_with_rows_in_8_bits(model_dirs, plain_models, name):
    """Against the plain implementation with its rows rounded where the engine rounds them. What differs by bfloat16's rounding (2^-9 of a value) may fall to another e4m3
    number (steps of 2^-3 to 2^-4): one value in 16 to 32 by up to 2^-3, 2^-3 / sqrt(24) = 2.6 % of a row in the 2-norm at most and a third of that where steps
    are uniform; four products a layer, three layers: 2.6 % / 3 * sqrt(12) = 3 % of the residual's share, 6 % of the largest logit allowed."""
    config, tensors = plain_models[name]
    mine = rounded(tensors, plan_of(config), through_bf16=True)
    mine = {k: (plain.round_to_bf16(v) if v.ndim >= 2 and ("wte" in k or "wpe" in k) else v) for k, v in mine.items()}
    V = config["vocab_size"]
    reqs = {f"r{i}": tt.random_tokens(40 + i, n, V) for i, n in enumerate([70, 21, 1, 100])}
    ref = {rid: forward_rows8(config, mine, toks) for rid, toks in reqs.items()}
    for label, make in SCHEDULES.items():
        steps = make(reqs)
        core = core_of(model_dirs[name], steps, weights="mxfp4", rows="mxfp8")
        got = tt.run_schedule(core, steps)
        tt.check_against_plain(got, reqs, ref, 6e-2, f"mxfp8 {name} {label}", family="GPT-2 with rows in 8 bits")
        del core


LARULORN = {"architecture": "Larulorn", "vocab": 300, "width": 64, "norm": {"eps": 1e-5}, "logit_scale": 0.75, "layers": [
    {"type": "attention", "mixer": {"heads": 4, "kv_heads": 2, "dim": 16, "vdim": 16, "scale": 0.25, "v_mix": True, "rot": {"dims": 8, "base": 10000.0}}, "mlp": {"kind": "dense", "ff": 104, "limit": 7.0}},
    {"type": "attention", "mixer": {"heads": 4, "kv_heads": 2, "dim": 16, "vdim": 16, "scale": 0.18, "v_mix": True}, "mlp": {"kind": "dense", "ff": 80, "limit": 2.0}}]}
LAFANEX = {"architecture": "Lafanex", "vocab": 300, "width": 64, "norm": {"eps": 1e-5}, "layers": [
    {"type": "attention", "mixer": {"heads": 4, "kv_heads": 2, "dim": 16, "vdim": 16, "scale": 0.3, "rot": {"dims": 8, "base": 10000.0}}, "mlp": {"kind": "dense", "ff": 96}},
    {"type": "mamba1", "mixer": {"inner": 128, "state": 16, "dt_rank": 4, "conv": 4}, "mlp": {"kind": "dense", "ff": 72}},
    {"type": "mamba1", "mixer": {"inner": 96, "state": 8, "dt_rank": 6, "conv": 3}, "mlp": None}]}
DESIGNS = {"larulorn": (LARULORN, plain_larulorn), "lafanex": (LAFANEX, plain_lafanex), "lafanex_streams": (dict(LAFANEX, streams=2), plain_lafanex)}


@pytest.fixture(scope="module")
def designs(tmp_path_factory):
    from liyab_amd.weights import write_random_model

    out = {}
    for name, (config, module) in DESIGNS.items():
        d = str(tmp_path_factory.mktemp(name))
        write_random_model(d, config, 11)
        config, tensors = plain.read_model(d)
        out[name] = (d, config, tensors, module)
    return out


@pytest.mark.parametrize("name", sorted(DESIGNS))
def test_designs_in_4_bits(designs, name):
    """The 32-bit path over rounded matrices, as the unrounded designs are tested."""
    d, config, tensors, module = designs[name]
    mine = rounded(tensors, plan_of(config))
    reqs = {f"r{i}": tt.random_tokens(60 + i, n, config["vocab"]) for i, n in enumerate([40, 13, 1, 66])}
    ref = {rid: module.forward(config, mine, toks) for rid, toks in reqs.items()}
    for label, make in SCHEDULES.items():
        steps = make(reqs)
        got = tt.run_schedule(core_of(d, steps, "float32", weights="mxfp4"), steps)
        tt.check_against_plain(got, reqs, ref, TOL["float32"], f"mxfp4 {name} {label}", family="designs in 4 bits, float32")


def rms_off(got, want):
    a, b = (np.concatenate([g[rid][p] for rid in sorted(g) for p in sorted(g[rid])]).astype(np.float64) for g in (got, want))
    return float(np.linalg.norm(a - b) / np.linalg.norm(b))


@pytest.mark.parametrize("name", sorted(DESIGNS))
def test_designs_with_rows_in_8_bits(designs, name):
    """Beside rows in bfloat16 over the same matrices: e4m3 rounds a value by up to 2^-4 of it, 2^-4 / sqrt(3) in the mean, each of at most 12 products: 12.5 % in the
    2-norm at most, and not the same."""
    d, config, _, _ = designs[name]
    reqs = {f"r{i}": tt.random_tokens(60 + i, n, config["vocab"]) for i, n in enumerate([40, 13, 1, 66])}
    for label, make in SCHEDULES.items():
        steps = make(reqs)
        wide = tt.run_schedule(core_of(d, steps, weights="mxfp4"), steps)
        got = tt.run_schedule(core_of(d, steps, weights="mxfp4", rows="mxfp8"), steps)
        off = rms_off(got, wide)
        assert 1e-4 < off < 0.125, f"{name} {label}: {off}"


@pytest.mark.parametrize("rows", [None, "mxfp8"])
def test_replies_do_not_depend_on_the_batch(model_dirs, plain_models, rows):
    """batch_invariant: the same bits however the tokens are cut into steps and whatever else a step holds."""
    config, _ = plain_models["B"]
    reqs = {f"i{i}": tt.random_tokens(500 + i, n, config["vocab_size"]) for i, n in enumerate([150, 33, 9, 70, 200])}
    runs = {}
    for label, steps in (("whole", tt.schedule_whole(reqs)), ("tail", tt.schedule_bulk_tail(reqs, tail=12)), ("mixed", tt.schedule_mixed(reqs, seed=4, decode_tail=10))):
        core = core_of(model_dirs["B"], steps, batch_invariant=True, weights="mxfp4", rows=rows)
        runs[label] = tt.run_schedule(core, steps)
        assert core.step_fn.graph_replays > 0 or label == "whole"
        del core
    for label in ("tail", "mixed"):
        for rid, toks in reqs.items():
            for p in range(len(toks)):
                assert np.array_equal(runs[label][rid][p], runs["whole"][rid][p]), f"{label}: request {rid} position {p}"


def test_layers_run_from_one_recorded_list(tmp_path):
    """Layers after the first of their kind run natively from its launches, their own 4-bit matrices among the addresses."""
    from liyab_amd.weights import write_random_model

    write_random_model(str(tmp_path), dict(CONFIG_A, n_layer=5), 3)
    config, tensors = plain.read_model(str(tmp_path))
    reqs = {"a": tt.random_tokens(1, 50, config["vocab_size"]), "b": tt.random_tokens(2, 30, config["vocab_size"])}
    steps = tt.schedule_whole(reqs)
    for rows in (None, "mxfp8"):
        core = core_of(str(tmp_path), steps, weights="mxfp4", rows=rows)
        got = tt.run_schedule(core, steps)
        assert core.model.replayed_layers > 0
        core.model.replay_layers = False
        again = tt.run_schedule(core, steps)
        for rid, toks in reqs.items():
            for p in range(len(toks)):
                assert np.array_equal(got[rid][p], again[rid][p])


def test_memory_is_a_quarter(model_dirs):
    """What a matrix takes: 17 bytes for 32 values, whole blocks of 16 rows and 128 columns."""
    core = core_of(model_dirs["A"], [{"entries": [("a", [1, 2], [1])], "end": ["a"]}], weights="mxfp4")
    w = core.model.blocks[0].ffn.up_weight
    assert w.shape == (256, 64) and w.bytes() == 256 // 16 * 1 * 1088


def test_refusals(model_dirs):
    from liyab_amd import Engine
    from liyab_amd.engine import EngineCore
    from liyab_amd.errors import InvalidArgument, Unsupported

    d = model_dirs["A"]
    for kw in (dict(weights="int4"), dict(weights="mxfp4", rows="fp8"), dict(rows="mxfp8"), dict(weights="mxfp4", rows="mxfp8", dtype="float32")):
        with pytest.raises(InvalidArgument):
            EngineCore(d, page_size=16, max_tokens=256, **kw)
    core = EngineCore(d, page_size=16, max_tokens=256)
    with pytest.raises(InvalidArgument):
        Engine(core=core, weights="mxfp4")


def test_a_model_without_such_matrices_is_refused(tmp_path):
    from liyab_amd.engine import EngineCore
    from liyab_amd.errors import Unsupported
    from liyab_amd.weights import write_random_model

    m = {"heads": 4, "dim": 16, "vdim": 16, "kv_rank": 32, "scale": 0.25}
    write_random_model(str(tmp_path), {"architecture": "Bokulix", "vocab": 300, "width": 64, "max_positions": 256, "norm": {"eps": 1e-5},
                                       "layers": [{"type": "latent_attention", "mixer": m, "mlp": {"kind": "moe", "expert": {"ff": 64}, "router": {"experts": 8, "top": 2}}}]}, seed=1)
    with pytest.raises(Unsupported):
        EngineCore(str(tmp_path), page_size=16, max_tokens=256, weights="mxfp4")


def test_generation_and_the_command_line(model_dirs):
    """The public engine, greedy, the same tokens from the command line."""
    from liyab_amd import Engine, SamplingParams

    engine = Engine(model_dirs["A"], weights="mxfp4", rows="mxfp8", page_size=16, num_pages=32, max_num_seqs=4)
    engine.stop_at_eos = False
    want = engine.generate([5, 17, 3], SamplingParams(temperature=0.0, max_tokens=12)).tokens
    assert len(want) == 12
    del engine
    r = subprocess.run([sys.executable, "-m", "liyab_amd.cli", "-m", model_dirs["A"], "-p", "5,17,3", "-n", "12", "--temp", "0", "--weights", "mxfp4", "--rows", "mxfp8"],
                       capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stderr[-2000:]
    assert [int(t) for t in r.stdout.replace(",", " ").split()] == want


def test_loading_holds_one_wide_matrix_at_a_time(tmp_path):
    """A model that fits the device's memory in 4 bits loads there: what is allocated on the way stays under the 4-bit model, the tables and one matrix, as it is stored (4 bytes) and as
    it is rounded (2, and 2 more where it is stored the other way round)."""
    from liyab_amd.models.loading import load_model
    from liyab_amd.weights import write_random_model

    width, layers, vocab = 512, 6, 64
    config = dict(CONFIG_A, n_layer=layers, n_embd=width, n_head=8, vocab_size=vocab, n_positions=128)
    write_random_model(str(tmp_path), config, 5)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    _, model = load_model(str(tmp_path), "bfloat16", "cuda:0", weights="mxfp4")
    values = 12 * width * width * layers
    peak = torch.cuda.max_memory_allocated() - before
    assert peak < values * 17 // 32 + 4 * width * width * 8 + (vocab + 128) * width * 8 + (1 << 20), f"{peak} bytes on the way, the wide matrices are {2 * values}"
    one, other = model.blocks[0].ffn, model.blocks[1].ffn
    assert one.up_weight is not other.up_weight


def test_the_same_matrix_is_kept_once(tmp_path):
    """By the names of what it is made of, and of the layout it is asked for in: not by where a wide matrix happens to lie."""
    from liyab_amd.config.plan import TensorSource
    from liyab_amd.parts.linear import product_matrix
    from liyab_amd.weights.loader import WeightStore

    w = {n: torch.randn(64, 64, generator=torch.Generator().manual_seed(i)) for i, n in enumerate("ab")}
    store = WeightStore(w, device="cuda:0", compute_dtype=torch.float32, products="mxfp4")
    a = product_matrix(store, TensorSource("a"), (64, 64))
    assert product_matrix(store, TensorSource("a"), (64, 64)) is a
    turned = product_matrix(store, TensorSource("a", layout="in_out"), (64, 64))
    doubled = product_matrix(store, TensorSource("a"), (64, 64), (("doubled", "a"), lambda m: 2 * m))
    joined = product_matrix(store, [TensorSource("a"), TensorSource("b")], [(64, 64)] * 2)
    from liyab_amd.kernels.mx import Mxfp4Matrix

    for got, wide in ((a, w["a"]), (turned, w["a"].t()), (doubled, 2 * w["a"]), (joined, torch.cat([w["a"], w["b"]]))):
        assert torch.equal(got.blocks, Mxfp4Matrix.quantize(wide.contiguous().to("cuda:0")).blocks)
    assert not store._cache and not store._derived
