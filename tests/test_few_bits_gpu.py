"""A whole model served in few bits against the plain implementation with its keys and values rounded as the cache rounds them and its
matrices as the weights are.

Tolerances (of the largest logit). float32: 2e-5 for the order of sums, and what follows from a payload of the first layer that rounds the other
way because two float32 orders of arithmetic straddle a tie (values differ by about 2^-22 of them and ties lie 2^-4 apart, so one payload in
2^17 or so: about one in three requests of 90 tokens, and the first layer's are counted below). One step of e4m3, 2^-4 of one of 64 features of a key or value,
moves the stream by about e = 1e-3. The second layer's keys and values then differ by e, which moves e / 2^-4 = 1.6 % of its payloads by a step:
sqrt(0.016) 2^-4 = 8e-3 of a score or value, root mean square. Together 1e-3 + 8e-3. bfloat16: the replay tests' 2e-2, and as much again because a
key's 2^-8 moves one payload in sixteen to its neighbour."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import plain_e4m3
import plain_qwen3 as plain
import replay_util as R
from tiny_configs import _config
from vosti_b200 import Engine, ops
from vosti_b200.engine.batch import StepEntry
from vosti_b200.weights import write_random_model

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]
TOLERANCE = {"float32": 9.02e-3, "bfloat16": 4e-2}
CONFIGS = {
    "d64": _config(num_hidden_layers=2, hidden_size=128, num_attention_heads=4, num_key_value_heads=2, head_dim=64, intermediate_size=192, vocab_size=300,
                   rope_theta=10000.0, rms_norm_eps=1e-6, tie_word_embeddings=True, max_position_embeddings=512),
    "d128": _config(num_hidden_layers=2, hidden_size=200, num_attention_heads=5, num_key_value_heads=1, head_dim=128, intermediate_size=320, vocab_size=256,
                    rope_theta=1000000.0, rms_norm_eps=1e-5, tie_word_embeddings=False, max_position_embeddings=512),
    "d48": _config(num_hidden_layers=2, hidden_size=80, num_attention_heads=6, num_key_value_heads=3, head_dim=48, intermediate_size=200, vocab_size=331,
                   rope_theta=50000.0, rms_norm_eps=3e-6, tie_word_embeddings=False, max_position_embeddings=640),
}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    out = {}
    for seed, (name, config) in enumerate(CONFIGS.items()):
        folder = tmp_path_factory.mktemp(f"few_{name}")
        write_random_model(folder, config, seed + 3)
        out[name] = str(folder)
    return out


def in_four_bits(config, W, group):
    """The plain model's matrices as the engine rounds them: projections of q, k and v together, gate and up together."""
    W = dict(W)
    for i in range(config["num_hidden_layers"]):
        p = f"model.layers.{i}."
        for names in ([f"self_attn.{n}_proj.weight" for n in "qkv"], ["self_attn.o_proj.weight"], ["mlp.gate_proj.weight", "mlp.up_proj.weight"], ["mlp.down_proj.weight"]):
            whole = torch.cat([W[p + n] for n in names]).to(torch.bfloat16)
            numbers, at = ops.Int4Weight.quantize(whole, group).dequantized(), 0
            for n in names:
                rows = W[p + n].shape[0]
                W[p + n] = numbers[at:at + rows]
                at += rows
    return W


class Cache:
    """Keys or values of one layer and request [tokens, heads, d] as the cache holds them, step by step."""

    def __init__(self):
        self.rows, self.bytes = None, {}

    def add(self, new):
        start = 0 if self.rows is None else self.rows.shape[0]
        end = start + new.shape[0]
        self.rows = torch.zeros(end, *new.shape[1:], dtype=torch.float64) if self.rows is None else torch.cat([self.rows, torch.zeros_like(new, dtype=torch.float64)])
        to_payload = lambda x: x.float().clamp(-448, 448).to(torch.float8_e4m3fn).double()
        for block in range(start // 16, (end - 1) // 16 + 1):
            lo, hi = max(start, block * 16), min(end, block * 16 + 16)
            for g in range(new.shape[1]):
                fresh = new[lo - start:hi - start, g].double()
                byte = plain_e4m3.scale_for(float(fresh.abs().max()))
                if lo % 16:
                    byte = max(byte, self.bytes[block, g])
                    self.rows[block * 16:lo, g] = to_payload(self.rows[block * 16:lo, g] * 2.0 ** (127 - byte)) * 2.0 ** (byte - 127)
                self.bytes[block, g] = byte
                self.rows[lo:hi, g] = to_payload(fresh * 2.0 ** (127 - byte)) * 2.0 ** (byte - 127)
        return self.rows.float()


def logits_of_steps(config, W, steps, first=None):
    """Logits of every position of one request fed in `steps`; `first` (a list) receives the first layer's keys and values."""
    layers = config["num_hidden_layers"]
    caches = [(Cache(), Cache()) for _ in range(layers)]
    nq, nkv, d, eps = config["num_attention_heads"], config["num_key_value_heads"], config["head_dim"], config["rms_norm_eps"]
    out, start = [], 0
    for tokens in steps:
        positions = torch.arange(start, start + len(tokens))
        hidden, residual = plain.embedding(torch.tensor(tokens), W["model.embed_tokens.weight"]), None
        for i in range(layers):
            p = f"model.layers.{i}."
            if residual is None:
                residual, normed = hidden, plain.rms_norm(hidden, W[p + "input_layernorm.weight"], eps)
            else:
                normed, residual = plain.add_rms_norm(hidden, residual, W[p + "input_layernorm.weight"], eps)
            a = p + "self_attn."
            q, k, v = ((normed @ W[a + f"{n}_proj.weight"].T).view(len(tokens), -1, d) for n in "qkv")
            cos, sin = plain.rope_tables(positions, d, config["rope_theta"])
            q = plain.apply_rope(plain.head_rms_norm(q, W[a + "q_norm.weight"], eps), cos, sin)
            k = plain.apply_rope(plain.head_rms_norm(k, W[a + "k_norm.weight"], eps), cos, sin)
            keys, values = (c.add(x).transpose(0, 1) for c, x in zip(caches[i], (k, v)))
            attn, _, _ = plain_e4m3.attend(q, keys, values, pos=positions, nq=nq, nkv=nkv, scale=d ** -0.5, window=0)
            normed, residual = plain.add_rms_norm(attn.float().reshape(len(tokens), nq * d) @ W[a + "o_proj.weight"].T, residual, W[p + "post_attention_layernorm.weight"], eps)
            hidden = plain.swiglu(normed, W[p + "mlp.gate_proj.weight"], W[p + "mlp.up_proj.weight"], W[p + "mlp.down_proj.weight"])
        final, _ = plain.add_rms_norm(hidden, residual, W["model.norm.weight"], eps)
        head = W["model.embed_tokens.weight"] if config["tie_word_embeddings"] else W["lm_head.weight"]
        out.append(final @ head.T)
        start += len(tokens)
    if first is not None:
        first.extend(c.rows for c in caches[0])
    return torch.cat(out)


def cut(tokens, sizes):
    out, at = [], 0
    for n in sizes:
        out.append(tokens[at:at + n])
        at += n
    return [s for s in out if s]


@pytest.mark.parametrize("name", sorted(CONFIGS))
@pytest.mark.parametrize("dtype,weights,group", [("float32", None, 128), ("bfloat16", None, 128), ("bfloat16", "int4", 64)])
@pytest.mark.parametrize("sizes", [[90], [33, 1, 1, 1, 20, 1], [5, 2, 9, 16, 17, 3, 1, 1], [1] * 40])
def test_logits(folders, name, dtype, weights, group, sizes):
    config, W = plain.load_model(folders[name])
    if weights:
        W = in_four_bits(config, W, group)
    engine = Engine(folders[name], dtype=dtype, num_blocks=64, max_num_seqs=4, cache_dtype="e4m3", weights=weights, weight_group=group)
    requests = {r: R.random_tokens(config["vocab_size"], sum(sizes), seed=17 + r) for r in range(3)}
    runner, got = engine.runner, {r: [] for r in requests}
    for r in requests:
        runner.begin(r)
    steps = {r: cut(tokens, sizes if r else [sum(sizes)]) for r, tokens in requests.items()}     # (the first request comes whole)
    for turn in range(len(sizes)):
        entries = [StepEntry(r, steps[r][turn], list(range(len(steps[r][turn])))) for r in requests if turn < len(steps[r])]
        logits, at = runner.step(entries).cpu(), 0
        for e in entries:
            got[e.request_id].append(logits[at:at + len(e.tokens)])
            at += len(e.tokens)
    runner.check_status()
    differ = 0
    held = plain_e4m3.dequantized(runner.cache.layer_caches[0].e4m3)
    for r in requests:
        first = []
        want, have = logits_of_steps(config, W, steps[r], first), torch.cat(got[r])
        at = torch.arange(sum(sizes))
        pages = torch.tensor(runner.cache.block_row(r, 0))[at // 16]
        differ += sum(int((have_[pages, :, at % 16] != want_).sum()) for have_, want_ in zip(held, first))
        worst = float((have - want).abs().max() / max(1.0, float(want.abs().max())))
        assert worst <= TOLERANCE[dtype], (r, worst)
    if dtype == "float32":
        assert differ <= 8, differ               # (of up to 69,120 payloads; one tie in 2^17 is straddled)


@pytest.mark.parametrize("weights", [None, "int4"])
def test_generation(folders, weights):
    """Graphs, scheduling ahead, portions, reused prefixes and preemption: greedy tokens are the same, and the plain model's choice."""
    name = "d64"
    config, W = plain.load_model(folders[name])
    prompts = [R.random_tokens(config["vocab_size"], n, seed=n) for n in (5, 40, 33, 70)]
    common = dict(dtype="bfloat16", max_num_seqs=4, cache_dtype="e4m3", weights=weights, weight_group=32)
    outputs = Engine(folders[name], num_blocks=128, cuda_graphs=False, **common).generate(prompts, max_tokens=24)
    engine = Engine(folders[name], num_blocks=128, async_scheduling=True, **common)
    assert engine.generate(prompts, max_tokens=24) == outputs
    assert engine.graphs.replays > 0
    engine.runner.cache.check()
    if weights:
        W = in_four_bits(config, W, 32)
    for prompt, out in zip(prompts, outputs):
        logits = logits_of_steps(config, W, [prompt] + [[t] for t in out[:-1]])[len(prompt) - 1:]
        for row, token in zip(logits, out):
            assert float(row.max() - row[token]) <= 2 * TOLERANCE["bfloat16"] * max(1.0, float(row.abs().max()))
    # a prompt whose start is in the cache already, and too few pages for all at once
    again = Engine(folders[name], num_blocks=128, **common)
    again.generate([prompts[3]], max_tokens=2)
    again.generate([prompts[3][:64] + prompts[0]], max_tokens=4)
    assert again.cache_stats()["reused_prefix_blocks"] >= 4
    tight = Engine(folders[name], num_blocks=12, enable_prefix_caching=False, **common)
    assert [len(o) for o in tight.generate(prompts, max_tokens=24)] == [24] * 4
    assert tight.cache_stats()["preemptions"] > 0
    tight.runner.cache.check()


def test_bytes(folders):
    """What is counted: 8 bits a key and value and a byte of scale for 16 tokens, 4 bits a weight and a scale a group."""
    wide, few = (Engine(folders["d64"], num_blocks=16, **kw) for kw in ({}, dict(cache_dtype="e4m3", weights="int4", weight_group=32)))
    assert wide.runner.cache.bytes_per_token() == 2 * 2 * 2 * 64 * 2
    assert few.runner.cache.bytes_per_token() == 2 * 2 * 2 * 64 + 1          # (8 scales for 16 tokens, rounded up)
    assert few.runner.model.weight_bytes() < 0.55 * wide.runner.model.weight_bytes()


def test_command_line(folders):
    run = lambda *more: subprocess.run([sys.executable, str(ROOT / "bin/vosti_engine_qwen3"), "--model", folders["d64"], "--prompt-ids", "5,6,7", "--max-tokens", "4",
                                        "--ignore-eos", *more], capture_output=True, text=True, timeout=600)
    few = run("--cache-dtype", "e4m3", "--weights", "int4", "--weight-group", "64")
    assert few.returncode == 0 and "MODEL_OUTPUT_TOKEN_IDS=[" in few.stdout, few.stderr[-2000:]
    refused = run("--cache-dtype", "e4m3", "--block-size", "8")
    assert refused.returncode != 0 and "multiple of 16" in refused.stderr


def test_layers_that_read_another_layers_cache(folders):
    """A run order in which a layer reads the keys and values, in 8 bits, of the one before it."""
    import dataclasses
    from vosti_b200.config import RunEntry, model_spec_from_dir
    from vosti_b200.weights import load_weights
    from vosti_b200.models import build_model
    spec = dataclasses.replace(model_spec_from_dir(folders["d64"]), run_order=(RunEntry(0), RunEntry(1, cache_from=0)))
    tensors = load_weights(folders["d64"], build_model(spec).expected_weights(), device=torch.device("cuda:0"), dtype=torch.bfloat16, ignore=build_model(spec).ignorable_weights(),
                           aliases=build_model(spec).tied_weights())
    tokens = R.random_tokens(300, 60, seed=1)
    got = []
    for cache in (None, "e4m3"):
        engine = Engine(spec=spec, tensors=dict(tensors), num_blocks=16, cache_dtype=cache)
        engine.runner.begin(0)
        rows = [engine.runner.step([StepEntry(0, tokens[:50], [49])])] + [engine.runner.step([StepEntry(0, [t], [0])]) for t in tokens[50:]]
        engine.runner.check_status()
        got.append(torch.cat(rows).cpu())
    # (keys and values of 8 bits: 2^-4 of each at most, some 2^-5 / sqrt(3) of it on the average)
    assert float((got[0] - got[1]).abs().max() / got[0].abs().max()) < 0.25 and not torch.equal(got[0], got[1])
