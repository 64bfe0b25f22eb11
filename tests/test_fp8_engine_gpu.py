"""The engine with its layers' matrices held in 8 bits."""
import pytest
import torch

import fp8_plain as P8
import helpers as H

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def _runner(d, weights="fp8", page_size=16, pages=64, **env):
    from binfer_b200.engine import make_env, make_runner
    from binfer_b200.engine.loading import model_from_dir
    env = make_env("bfloat16", weights=weights, **env)
    return make_runner(model_from_dir(d, env), env, page_size=page_size, num_pages=pages)


@pytest.mark.parametrize("which", ["M", "O"])
def test_weights_are_the_checkpoint_s_in_8_bits(cuda_device, tmp_path, which):
    d = H.make_model_dir(tmp_path, which, BF16)
    raw, w = H.read_model_dir(d)
    w = {n: t.to(BF16).to(cuda_device) for n, t in w.items()}
    for i, b in enumerate(_runner(d).model.blocks):
        a, m = f"model.layers.{i}.self_attn.", f"model.layers.{i}.mlp."
        for held, mats, gated in (
                (b.mixer.w_qkv, [w[a + f"{n}_proj.weight"] for n in "qkv"], False),
                (b.mixer.w_o, [w[a + "o_proj.weight"]], False),
                (b.ffn.w_gate_up, [w[m + "gate_proj.weight"], w[m + "up_proj.weight"]], True),
                (b.ffn.w_out, [w[m + "down_proj.weight"]], False)):
            codes, scales = P8.hold_weight(torch.cat(mats), gated)
            assert torch.equal(held.codes.to(F32).to(F64), codes) and torch.equal(held.scales, scales)


@pytest.mark.parametrize("which,kv_cache", [("M", "auto"), ("M", "int4"), ("V", "auto")])
def test_every_product_of_a_step(cuda_device, tmp_path, monkeypatch, which, kv_cache):
    """Each product that the steps make (a prompt in portions, single tokens, both at once) is that of its
    inputs with the held weight; four a layer."""
    from binfer_b200.csrc import ops
    from binfer_b200.engine import StepItem
    d = H.make_model_dir(tmp_path, which, BF16)
    raw, _ = H.read_model_dir(d)
    runner = _runner(d, kv_cache=kv_cache)
    seen, whole = [], ops.fp8_linear

    def watched(x, w, out, **kw):
        whole(x, w, out, **kw)
        if isinstance(x, ops.Fp8Rows):         # (held numbers put into 8 bits once more are what they were)
            rows, x = x, torch.empty(x.shape, device=cuda_device)
            ops.fp8_rows_read(*rows, x)
        ref, off = P8.product(x, w.codes.to(F32).to(F64), w.scales, w.gated)
        diff = (out.to(F64) - ref).abs()
        assert (diff <= off + ref.abs() * (torch.finfo(out.dtype).eps / 2)).all()
        seen.append(tuple(w.shape))
    monkeypatch.setattr(ops, "fp8_linear", watched)
    ids = {"a": H.random_tokens(300, raw["vocab_size"], 3), "b": H.random_tokens(60, raw["vocab_size"], 4)}
    for rid in ids:
        runner.add_request(rid)
    for cut in ({"a": (0, 270)}, {"a": (270, 271), "b": (0, 40)}, {"a": (271, 272), "b": (40, 41)}):
        seen.clear()
        runner.step([StepItem(rid, ids[rid][a:b], [b - a - 1]) for rid, (a, b) in cut.items()])
        assert len(seen) == 4 * raw["num_hidden_layers"]
    runner.check_errors()


@pytest.mark.parametrize("which,kv_cache", [("M", "auto"), ("V", "int4"), ("O", "auto")])
def test_generation_with_and_without_graphs(cuda_device, tmp_path, which, kv_cache):
    from binfer_b200 import Engine
    d = H.make_model_dir(tmp_path, which, BF16)
    raw, _ = H.read_model_dir(d)
    prompts = [H.random_tokens(n, raw["vocab_size"], n) for n in (5, 190, 33, 1)]
    outs = []
    for graphs in (True, False, True):
        eng = Engine(d, "bfloat16", num_pages=96, max_seq_len=512, max_batch_size=4, cuda_graphs=graphs,
                     kv_cache=kv_cache, weights="fp8")
        outs.append(eng.generate(prompts, max_tokens=40, ignore_eos=True))
        if graphs:
            assert eng.runner.graph_replays > 0
    assert outs[0] == outs[1] == outs[2] and all(len(o) == 40 for o in outs[0])


def test_logits_are_near_those_of_the_other_engine(cuda_device, tmp_path):
    """A number in 8 bits is off by up to half of a step of 2^-3 to 2^-4 of itself, 0.0265 in the mean square;
    a product's sums, of independent errors of both factors, by sqrt(2) of that, 0.0375.  Two products one
    behind the other (values and output; gate, up and down, whose first two multiply) are off by at most
    0.0375 sqrt(4) = 0.075 of their size, and the error that a layer's input brings is passed on with a gain of
    about one.  Two sublayers in a row: sqrt(2) 0.075; the stream that they are added to does not lose."""
    from binfer_b200.engine import StepItem
    d = H.make_model_dir(tmp_path, "M", BF16)
    raw, _ = H.read_model_dir(d)
    ids = H.random_tokens(120, raw["vocab_size"], 5)
    got = []
    for weights in ("fp8", "auto"):
        r = _runner(d, weights)
        r.add_request("a")
        got.append(r.step([StepItem("a", ids, list(range(120)))]).double().cpu())
    off = H.rel_rms(*got)
    assert 1e-3 < off < 2 * 2 ** 0.5 * 0.075, off


def test_half_of_the_memory(cuda_device, tmp_path):
    d = H.make_model_dir(tmp_path, "M", BF16)
    models = [_runner(d, w).model for w in ("auto", "fp8")]
    matrices = sum(t.numel() for b in models[0].blocks
                   for t in (b.mixer.w_qkv, b.mixer.w_o, b.ffn.w_gate_up, b.ffn.w_out))
    saved = models[0].weight_bytes() - models[1].weight_bytes()
    # (a byte a number, less the scales and the rows' padding)
    assert 0.95 * matrices <= saved <= matrices


def test_what_is_refused(cuda_device, tmp_path):
    from binfer_b200 import Engine
    kw = dict(num_pages=16, max_seq_len=128, max_batch_size=2)
    m = H.make_model_dir(tmp_path, "M", BF16)
    with pytest.raises(ValueError, match="unknown weights"):
        Engine(m, "bfloat16", weights="int8", **kw)
    with pytest.raises(ValueError, match="bfloat16"):
        Engine(m, "float32", weights="fp8", **kw)
    with pytest.raises(ValueError, match="8 bits"):
        Engine(H.make_pabelix_dir(tmp_path / "p", "A", BF16), "bfloat16", weights="fp8", **kw)


def test_queries_alone(cuda_device, tmp_path):
    """A layer that reads another one's pages projects its queries only: the first rows of the stacked weight."""
    from binfer_b200.csrc import ops
    mixer = _runner(H.make_model_dir(tmp_path, "M", BF16)).model.blocks[0].mixer
    w, x = mixer._w_q(), torch.randn((7, mixer.hidden), device=cuda_device).to(BF16)
    out = torch.empty((7, mixer.q_size), dtype=BF16, device=cuda_device)
    ops.fp8_linear(x, w, out)
    ref, off = P8.product(x, mixer.w_qkv.codes[:mixer.q_size].to(F32).to(F64), mixer.w_qkv.scales[:w.scales.shape[0]])
    assert ((out.to(F64) - ref).abs() <= off + ref.abs() * 2.0 ** -8).all()


@pytest.mark.parametrize("norm", ["tanh_norm", "layernorm", "rmsnorm"])
@pytest.mark.parametrize("hidden", [256, 260])
def test_pre_norm_layers_of_every_norm(cuda_device, monkeypatch, norm, hidden):
    """Pre-norm layers whose norms are not RMS, and rows that the norm's kernel in 8 bits does not take (a width
    that is no multiple of eight): every product of a step is that of its inputs."""
    import dataclasses
    from binfer_b200.config.qwen3 import Qwen3Config
    from binfer_b200.config.specs import NormSpec
    from binfer_b200.csrc import ops
    from binfer_b200.engine import StepItem, make_env, make_runner
    from binfer_b200.engine.loading import model_from_seed
    raw = dict(architectures=["Qwen3ForCausalLM"], model_type="qwen3", num_hidden_layers=2, hidden_size=hidden,
               num_attention_heads=4, num_key_value_heads=2, head_dim=64, intermediate_size=384, vocab_size=200,
               rope_theta=1e4, rms_norm_eps=1e-6, tie_word_embeddings=False, max_position_embeddings=1024,
               hidden_act="silu", attention_bias=False)

    class Config:
        def to_spec(self):
            spec = Qwen3Config.from_dict(raw).to_spec()
            ns = NormSpec(kind=norm, eps=1e-5, bias_suffix=".b" if norm != "rmsnorm" else None)
            return dataclasses.replace(spec, final_norm=ns,
                                       layers=tuple(dataclasses.replace(l, norm=ns) for l in spec.layers))
    env = make_env("bfloat16", weights="fp8")
    runner = make_runner(model_from_seed(Config(), env, 3, std=0.06, norm_std=0.1), env, page_size=16, num_pages=32)
    seen, whole = [], ops.fp8_linear

    def watched(x, w, out, **kw):
        whole(x, w, out, **kw)
        seen.append(type(x))
        if isinstance(x, ops.Fp8Rows):
            rows, x = x, torch.empty(x.shape, device=cuda_device)
            ops.fp8_rows_read(*rows, x)
        ref, off = P8.product(x, w.codes.to(F32).to(F64), w.scales, w.gated)
        assert ((out.to(F64) - ref).abs() <= off + ref.abs() * (torch.finfo(out.dtype).eps / 2)).all()
    monkeypatch.setattr(ops, "fp8_linear", watched)
    ids = H.random_tokens(70, 200, 3)
    runner.add_request("a")
    for a, b in ((0, 60), (60, 61), (61, 70)):
        seen.clear()
        logits = runner.step([StepItem("a", ids[a:b], [b - a - 1])])
        assert len(seen) == 8 and torch.isfinite(logits).all()
        assert seen.count(ops.Fp8Rows) == (4 if norm == "rmsnorm" and hidden == 256 else 0)
    runner.check_errors()
