"""Every arrangement of layers with matrices in 4 bits: the designs' own configurations over rounded matrices, against their plain implementations."""

import json
import os
import shutil

import numpy as np
import pytest
import torch

import plain_mx
import test_dopilorn_gpu
import test_lafanex_gpu
import test_larulorn_gpu
import test_lolulorn_gpu
import test_mofulix_gpu
import trace_tools as tt
from conftest import TOL
from plain_gpt2 import read_model, round_to_bf16

pytestmark = pytest.mark.gpu

FAMILIES = {m.__name__.split("_")[1]: m for m in (test_dopilorn_gpu, test_lafanex_gpu, test_larulorn_gpu, test_lolulorn_gpu, test_mofulix_gpu)}

# what is rounded: the plan's spec kinds and the tensors that they read through products alone
IN_4_BITS = {"scored_attention": ("q", "k", "v", "gate", "out"), "clamped_glu": ("gate", "up", "down"), "gated_ffn": ("gate", "up", "down"),
             "normed_powers_ffn": ("up", "down"), "selective_scan": ("in", "out")}


def specs(plan):
    for layer in plan.layers:
        todo = [layer.mixer, layer.ffn]
        while todo:
            spec = todo.pop()
            if spec is not None:
                yield spec
                todo += [getattr(spec, side, None) for side in ("left", "right")]


def plan_of(config):
    from liyab_amd.config.registry import config_from_dict

    return config_from_dict(json.loads(json.dumps(config))).plan()


def sources(plan):
    """The rounded matrices, by name: (where each lies, the widths of a head's columns as the file has them and as the engine pads them, or None). And how many products a token goes
    through."""
    from liyab_amd.kernels import ops

    out, products = {}, 0
    for spec in specs(plan):
        kind = getattr(spec, "kind", "")
        keys = IN_4_BITS.get(kind, ())
        products += 2 * bool(keys)
        for k in keys:
            if spec.tensors.get(k) is None:
                continue
            heads = None
            if kind == "scored_attention" and k == "out" and spec.head_dim != spec.value_dim and not spec.gated and max(spec.head_dim, spec.value_dim) <= ops.ATTENTION_MAX_HEAD_DIM:
                heads = spec.value_dim, -(-max(spec.head_dim, spec.value_dim) // 8) * 8  # (groups of 32 run over the padded columns)
            out[spec.tensors[k].name] = spec.tensors[k], heads
    return out, products


CASES = [(family, name) for family, module in FAMILIES.items() for name, (config, *_) in module.CONFIGS.items() if sources(plan_of(config))[0]]


def test_every_arrangement_is_among_them():
    kinds, blocks = set(), set()
    for family, name in CASES:
        plan = plan_of(FAMILIES[family].CONFIGS[name][0])
        kinds |= {getattr(s, "kind", "") for s in specs(plan)}
        blocks |= {layer.arrangement for layer in plan.layers}
    assert kinds >= set(IN_4_BITS) | {"side_by_side"}
    assert blocks >= {"parallel", "parallel_pair", "post_norm_gated", "sandwich", "streams"}


def rounded(tensors, plan, through_bf16):
    out = {}
    for name, (src, heads) in sources(plan)[0].items():
        w = round_to_bf16(tensors[name]) if through_bf16 else tensors[name]
        w = w.T if src.layout == "in_out" else w
        rows = w.shape[0]
        if heads is not None:
            w = np.pad(w.reshape(rows, -1, heads[0]), ((0, 0), (0, 0), (0, heads[1] - heads[0]))).reshape(rows, -1)
        q = plain_mx.values(*plain_mx.quantize(w, plain_mx.E2M1, 2), plain_mx.E2M1)
        if heads is not None:
            q = q.reshape(rows, -1, heads[1])[:, :, : heads[0]].reshape(rows, -1)
        out[name] = q.T if src.layout == "in_out" else q
    return out


def requests(vocab):
    return {f"r{i}": tt.random_tokens(70 + i, n, vocab) for i, n in enumerate([40, 13, 1, 70])}


SCHEDULES = {"whole": tt.schedule_whole, "mixed": lambda reqs: tt.schedule_mixed(reqs, seed=3, decode_tail=9)}


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    from liyab_amd.weights import write_random_model

    out = {}
    for family, name in CASES:
        config, seed = FAMILIES[family].CONFIGS[name][:2]
        d = str(tmp_path_factory.mktemp(f"{family}_{name}"))
        write_random_model(d, json.loads(json.dumps(config)), seed)
        out[(family, name)] = (d,) + read_model(d)
    return out


def logits(d, steps, dtype, **kw):
    from liyab_amd.engine import EngineCore

    core = EngineCore(d, dtype=dtype, page_size=16, max_tokens=tt.max_live_tokens(steps), max_requests=8, **kw)
    got = tt.run_schedule(core, steps)
    del core
    return got


def rel(got, want):
    return float(np.abs(np.asarray(got, dtype=np.float64) - want).max() / np.abs(want).max())


@pytest.mark.parametrize("family,name", CASES)
def test_designs_in_4_bits(models, family, name):
    """The 32-bit path over the rounded matrices, within the tolerance of the design's own tests. A position whose logits the plain implementation itself moves k times as far as the
    median one's, when every matrix moves by 2^-20 of its values, is allowed k times the tolerance: one token of a mixer that norms what nearly cancels is ten times as
    sensitive as the others, with wide matrices too."""
    module = FAMILIES[family]
    d, config, tensors = models[(family, name)]
    mine = {**tensors, **rounded(tensors, plan_of(module.CONFIGS[name][0]), False)}
    rng = np.random.default_rng(0)
    shaken = {k: v * (1 + 2.0 ** -20 * rng.choice([-1, 1], size=v.shape)) if v.ndim == 2 else v for k, v in mine.items()}
    reqs = requests(config["vocab"])

    def forward(weights):
        return {rid: module.plain.forward(toks, weights, config) if family == "dopilorn" else module.plain.forward(config, weights, toks) for rid, toks in reqs.items()}

    ref, other = forward(mine), forward(shaken)
    moved = {rid: [rel(other[rid][p], ref[rid][p]) for p in range(len(toks))] for rid, toks in reqs.items()}
    median = float(np.median(sum(moved.values(), [])))
    for label, make in SCHEDULES.items():
        got = logits(d, make(reqs), "float32", weights="mxfp4")
        for rid, toks in reqs.items():
            assert sorted(got[rid]) == list(range(len(toks)))
            for p in range(len(toks)):
                e, allowed = rel(got[rid][p], ref[rid][p]), TOL["float32"] * max(1.0, moved[rid][p] / median)
                assert e <= allowed, f"{family} {name} {label}: request {rid}, position {p}: {e} of {allowed}"


@pytest.mark.parametrize("family,name", CASES)
def test_designs_in_4_bits_beside_wide_matrices_of_their_values(models, family, name, tmp_path):
    """In bfloat16, which holds a 4-bit matrix's values exactly, the same model with wide matrices: products are the same numbers, only their sums are added in other orders. The
    tolerance of the design's own tests (root mean squares), and most positions far below it: a bfloat16 that falls the other way here and there."""
    from liyab_amd.weights.safetensors_io import write_safetensors

    module = FAMILIES[family]
    d, config, tensors = models[(family, name)]
    wide = {k: torch.tensor(v).float() for k, v in {**tensors, **rounded(tensors, plan_of(module.CONFIGS[name][0]), True)}.items()}
    shutil.copy(os.path.join(d, "config.json"), tmp_path)
    write_safetensors(str(tmp_path / "model.safetensors"), wide)
    reqs = requests(config["vocab"])
    for label, make in SCHEDULES.items():
        steps = make(reqs)
        got, ref = logits(d, steps, "bfloat16", weights="mxfp4"), logits(str(tmp_path), steps, "bfloat16")
        off = []
        for rid in reqs:
            for p in sorted(ref[rid]):
                a, b = (np.asarray(g[rid][p], dtype=np.float64) for g in (got, ref))
                off.append(float(np.sqrt(np.mean((a - b - (a - b).mean()) ** 2) / np.mean((b - b.mean()) ** 2))))
        assert max(off) <= module.TOL_B["bfloat16"] and np.median(off) <= module.TOL_B["bfloat16"] / 4, f"{family} {name} {label}: {max(off)}, median {np.median(off)}"


@pytest.mark.parametrize("family,name", CASES)
def test_designs_with_rows_in_8_bits(models, family, name):
    """Beside rows in bfloat16 over the same matrices: e4m3 rounds a value by up to 2^-4 of it, 2^-4 / sqrt(3) in the mean, at each of a token's products, and no product's input goes
    through a power above the third behind it. Routed layers' choices may fall differently: there, numbers."""
    d, config, _ = models[(family, name)]
    plan = plan_of(FAMILIES[family].CONFIGS[name][0])
    kinds = {getattr(s, "kind", "") for s in specs(plan)}
    bound = 2.0 ** -4 / 3 ** 0.5 * sources(plan)[1] ** 0.5 * (3 if "normed_powers_ffn" in kinds else 1)
    reqs = requests(config["vocab"])
    for label, make in SCHEDULES.items():
        steps = make(reqs)
        wide, got = logits(d, steps, "bfloat16", weights="mxfp4"), logits(d, steps, "bfloat16", weights="mxfp4", rows="mxfp8")
        a, b = (np.concatenate([g[rid][p] for rid in sorted(g) for p in sorted(g[rid])]).astype(np.float64) for g in (got, wide))
        assert np.isfinite(a).all() and not np.array_equal(a, b)
        if not any("routed" in k for k in kinds):
            off = float(np.linalg.norm(a - b) / np.linalg.norm(b))
            assert off < bound, f"{family} {name} {label}: {off} of {bound}"
