"""The engine with its cache held in 4 bits."""
import pytest
import torch

import helpers as H
import kv4_plain as K4
import qwen3_plain as P

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _runner(d, kv_cache, page_size=16, pages=64, **kw):
    from binfer_b200.engine import make_env, make_runner
    from binfer_b200.engine.loading import model_from_dir
    env = make_env("bfloat16", kv_cache=kv_cache)
    return make_runner(model_from_dir(d, env), env, page_size=page_size, num_pages=pages, **kw)


def _plain(monkeypatch, raw, w, ids, held):
    """Whole-sequence logits in double, keys and values as projected or as held in 4 bits."""
    whole = P.causal_attention
    with monkeypatch.context() as m:
        if held:
            m.setattr(P, "causal_attention", lambda q, k, v, scale, window=None: whole(
                q, K4.held(k.to(BF16)).to(k.dtype), K4.held(v.to(BF16)).to(v.dtype), scale, window))
        return P.forward(raw, {n: t.to(BF16) for n, t in w.items()}, ids, dtype=torch.float64)


@pytest.mark.parametrize("which,page_size", [("M", 16), ("M", 128), ("V", 16), ("O", 64)])
def test_cached_tokens_are_the_other_engine_s_in_4_bits(cuda_device, tmp_path, which, page_size):
    """The first layer's keys and values, of a prompt in portions and single tokens, are those of the
    engine with bfloat16 pages, held in 4 bits: every number."""
    from binfer_b200.engine import StepItem
    d = H.make_model_dir(tmp_path, which, BF16)
    raw, _ = H.read_model_dir(d)
    ids = H.random_tokens(143, raw["vocab_size"], 7)
    runners = [_runner(d, kv, page_size) for kv in ("auto", "int4")]
    for r in runners:
        r.add_request("a")
        for a, b in ((0, 37), (37, 140), (140, 141), (141, 142), (142, 143)):
            r.step([StepItem("a", ids[a:b], [b - a - 1])])
        r.check_errors()
    k, v = runners[0].views[0].k_cache, runners[0].views[0].v_cache
    k4, v4 = K4.unpack(runners[1].views[0].k_cache)
    assert runners[1].views[0].v_cache is None
    tables = [r.cache.get("a").tables[r.views[0].group] for r in runners]
    kept = 143 - (raw.get("sliding_window") or 143) if which == "V" else 0
    seen = 0
    for i, (p, p4) in enumerate(zip(*tables)):
        n = min(page_size, 143 - i * page_size)
        if p < 0 or n <= 0 or (i + 1) * page_size <= kept:
            continue
        assert torch.equal(K4.held(k[p, :, :n]).cpu(), k4[p4, :, :n])
        assert torch.equal(K4.held(v[p, :, :n]).cpu(), v4[p4, :, :n])
        seen += n
    assert seen >= 100


@pytest.mark.parametrize("which", ["M", "V", "F"])
def test_logits_follow_the_model_over_held_tokens(cuda_device, tmp_path, monkeypatch, which):
    """Prompts in portions, single tokens and both in one step.  The engine's keys and values differ from
    double ones by bfloat16 roundings, some 2^-9 of their size where a code's step is a third of it or
    less: some 2 % of the codes move by a step, which adds sqrt(0.02 * 12) = 0.5 of the error that holding
    them in 4 bits makes by itself (a step / sqrt(12)).  So the logits lie within 0.75 of the distance
    between the model over held tokens and the model over its own, and the engine's bfloat16 bound."""
    from binfer_b200.engine import StepItem
    d = H.make_model_dir(tmp_path, which, BF16)
    raw, w = H.read_model_dir(d)
    seqs = {"a": H.random_tokens(211, raw["vocab_size"], 3), "b": H.random_tokens(60, raw["vocab_size"], 4)}
    runner = _runner(d, "int4")
    for rid in seqs:
        runner.add_request(rid)
    got = {rid: [] for rid in seqs}
    cuts = [{"a": (0, 70)}, {"a": (70, 200), "b": (0, 1)}, {"a": (200, 201), "b": (1, 58)},
            {"a": (201, 202), "b": (58, 59)}, {"a": (202, 211), "b": (59, 60)}]
    for cut in cuts:
        items = [StepItem(rid, seqs[rid][a:b], list(range(b - a))) for rid, (a, b) in cut.items()]
        logits = runner.step(items).double().cpu()
        at = 0
        for rid, (a, b) in cut.items():
            got[rid].append(logits[at:at + b - a])
            at += b - a
    runner.check_errors()
    for rid, ids in seqs.items():
        held = _plain(monkeypatch, raw, w, ids, True)
        own = _plain(monkeypatch, raw, w, ids, False)
        off = H.rel_rms(torch.cat(got[rid]), held)
        assert off <= 0.75 * H.rel_rms(own, held) + 1.2e-2, off


@pytest.mark.parametrize("which,page_size", [("M", 16), ("V", 8), ("O", 32)])
def test_generation_with_and_without_graphs(cuda_device, tmp_path, which, page_size):
    """The same tokens from captured and eager decode steps, twice, and every page given back."""
    from binfer_b200 import Engine
    d = H.make_model_dir(tmp_path, which, BF16)
    raw, _ = H.read_model_dir(d)
    prompts = [H.random_tokens(n, raw["vocab_size"], n) for n in (5, 190, 33, 1)]
    outs = []
    for graphs in (True, False, True):
        eng = Engine(d, "bfloat16", num_pages=96, page_size=page_size, max_seq_len=512, max_batch_size=4,
                     cuda_graphs=graphs, kv_cache="int4")
        outs.append(eng.generate(prompts, max_tokens=40, ignore_eos=True))
        assert eng.stats()["pages_free"] == eng.stats()["pages_total"]
        if graphs:
            assert eng.runner.graph_replays > 0
    assert outs[0] == outs[1] == outs[2] and all(len(o) == 40 for o in outs[0])


def test_preemption(cuda_device, tmp_path):
    """Pages run out: a request is recomputed from its tokens, and all finish."""
    from binfer_b200 import Engine
    d = H.make_model_dir(tmp_path, "M", BF16)
    raw, _ = H.read_model_dir(d)
    eng = Engine(d, "bfloat16", num_pages=14, page_size=16, max_seq_len=160, max_batch_size=4, kv_cache="int4")
    outs = eng.generate([H.random_tokens(40, raw["vocab_size"], n) for n in range(4)], max_tokens=60,
                        ignore_eos=True)
    assert all(len(o) == 60 for o in outs) and eng.stats()["preemptions"] > 0


def test_a_page_takes_9_bits_where_it_took_32(cuda_device, tmp_path):
    from binfer_b200 import Engine
    d = H.make_model_dir(tmp_path, "M", BF16)
    kw = dict(max_kv_memory_gb=0.004, page_size=16, max_seq_len=65536, max_batch_size=64, cuda_graphs=False)
    pages = [Engine(d, "bfloat16", kv_cache=kv, **kw).runner.cache for kv in ("auto", "int4")]
    assert 3.5 < pages[1].num_pages / pages[0].num_pages < 3.6
    assert pages[1].storage_bytes() <= 0.004 * 2 ** 30 * 1.02


def test_what_is_refused(cuda_device, tmp_path):
    from binfer_b200 import Engine
    kw = dict(num_pages=16, max_seq_len=128, max_batch_size=2)
    m = H.make_model_dir(tmp_path, "M", BF16)
    for bad, match in ((dict(kv_cache="fp8"), "kv_cache"), (dict(kv_cache="int4", page_size=4), "pages"),
                       (dict(kv_cache="int4", page_size=48), "pages")):
        with pytest.raises(ValueError, match=match):
            Engine(m, "bfloat16", **dict(kw, **bad))
    with pytest.raises(ValueError, match="bfloat16"):
        Engine(m, "float32", kv_cache="int4", **kw)
    with pytest.raises(ValueError, match="heads"):
        Engine(H.make_model_dir(tmp_path / "b", "B", BF16), "bfloat16", kv_cache="int4", **kw)
    with pytest.raises(ValueError, match="4 bits"):
        Engine(H.make_pabelix_dir(tmp_path / "p", "A", BF16), "bfloat16", kv_cache="int4", **kw)
