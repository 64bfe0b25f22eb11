"""Captured decode steps described on the device: the same batch descriptions and tokens as from the host."""
import pytest
import torch

import helpers as H

pytestmark = pytest.mark.gpu


def _pair(tmp_path, monkeypatch, **kw):
    """Two runners over the same model, described from the device and from the host."""
    from binfer_b200.engine import make_env, make_runner, runner
    from binfer_b200.engine.loading import model_from_dir
    d = H.make_model_dir(tmp_path, "M", torch.bfloat16)
    env = make_env("bfloat16")
    model = model_from_dir(d, env)
    out = []
    for on in (True, False):
        r = make_runner(model, env, **kw)
        step = r._graph_step

        def run(*a, step=step, on=on, **k):
            monkeypatch.setattr(runner, "STEP_TABLES", on)
            return step(*a, **k)

        r._graph_step = run
        r.enable_decode_graphs(max_batch=4, max_seq_len=700)
        out.append(r)
    return out


def test_descriptions_and_logits_agree(cuda_device, tmp_path, monkeypatch):
    """Requests that come and go, portions between single tokens, a request whose slot and pages another
    takes over, a batch taken back by a token, tables that grow."""
    from binfer_b200.engine import StepItem
    dev, host = _pair(tmp_path, monkeypatch, page_size=16, num_pages=90, max_requests=4)
    toks = H.random_tokens(2000, 500, 1)

    def both(items):
        a, b = dev.step(items).clone(), host.step(items).clone()
        assert torch.equal(a, b)
        return a

    def single(rids):
        both([StepItem(r, [toks[ord(r) + dev.cache.get(r).length]], [0]) for r in rids])
        n = next(b for b in dev._buckets if b >= len(rids))
        d, h = dev._graphs[n], host._graphs[n]
        c = d["ctx"]
        f, _ = host._layout(n, n, n, [44])
        view = lambda name: h["dev"][f[name][0]:f[name][0] + f[name][1]]
        for name, t in (("token_ids", c.token_ids), ("positions", c.positions), ("seq_of_token", c.seq_of_token),
                        ("q_start", c.q_start), ("ctx_lens", c.ctx_lens), ("state_slots", c.state_slots),
                        ("logit_rows", c.logit_rows), ("slots0", c.slots[0]), ("tables0", c.block_tables[0].flatten())):
            assert torch.equal(t, view(name)), name

    for r in (dev, host):
        for rid in "abc":
            r.add_request(rid)
    both([StepItem("a", toks[:300], [299]), StepItem("b", toks[:5], [4])])
    for _ in range(20):
        single("ab")
    both([StepItem("c", toks[:33], [32]), StepItem("a", toks[7:9], [1])])
    for i in range(17):
        single("cab" if i % 2 else "ca")
    for r in (dev, host):
        r.free_request("a")
        r.add_request("d")
        r.add_request("e")
    both([StepItem("d", toks[:200], [199]), StepItem("e", toks[:1], [0])])
    for i in range(35):
        single("dbec")
        if i == 9:                                    # taken back, like a draft that is rejected
            for r in (dev, host):
                for rid in "dbec":
                    r.cache.get(rid).length -= 1
    for r in (dev, host):                             # wider tables
        r.enable_decode_graphs(max_batch=4, max_seq_len=700)
    single("be")
    dev.check_errors()


def test_what_a_refused_step_leaves(cuda_device, tmp_path, monkeypatch):
    """A step refused for want of ids changes nothing that the next one reads."""
    from binfer_b200.engine import StepItem
    dev, host = _pair(tmp_path, monkeypatch, page_size=16, num_pages=60, max_requests=2)
    for r in (dev, host):
        r.add_request("a")
        r.step([StepItem("a", list(range(31)), [30])])
        r.step([StepItem("a", [7], [0])])
        with pytest.raises(ValueError, match="device"):
            r.step([StepItem("a", [0], [0], src_row=0)])
    for t in range(20):
        assert torch.equal(dev.step([StepItem("a", [t], [0])]), host.step([StepItem("a", [t], [0])]))
    dev.check_errors()


@pytest.mark.parametrize("which", ["M", "O"])
def test_generation(cuda_device, tmp_path, monkeypatch, which):
    from binfer_b200 import Engine
    from binfer_b200.engine import runner
    d = H.make_model_dir(tmp_path, which, torch.bfloat16)
    raw, _ = H.read_model_dir(d)
    prompts = [H.random_tokens(n, raw["vocab_size"], n) for n in (3, 100, 47, 12, 61)]
    outs = []
    for on in (True, False):
        monkeypatch.setattr(runner, "STEP_TABLES", on)
        eng = Engine(d, "bfloat16", num_pages=40, page_size=16, max_seq_len=256, max_batch_size=4)
        outs.append(eng.generate(prompts, max_tokens=50, ignore_eos=True))
        assert eng.runner.graph_replays > 0
    assert outs[0] == outs[1]


def test_capture_with_an_engine_gone(cuda_device, tmp_path):
    """An engine that only a reference cycle holds is not collected in the middle of another's capture."""
    import gc
    from binfer_b200 import Engine
    d = H.make_model_dir(tmp_path, "M", torch.bfloat16)

    def engine():
        e = Engine(d, "bfloat16", num_pages=40, page_size=16, max_seq_len=256, max_batch_size=4)
        return e, e.generate([[1, 2, 3]], max_tokens=4, ignore_eos=True)

    was = gc.get_threshold()
    gc.collect()
    gc.disable()
    try:
        old, want = engine()
        old.itself = old
        del old
        new = Engine(d, "bfloat16", num_pages=40, page_size=16, max_seq_len=256, max_batch_size=4)
        forward, calls = new.model.forward, []

        def collecting(*a, **k):                  # the second forward is the captured one
            calls.append(gc.isenabled())
            if gc.isenabled() and torch.cuda.is_current_stream_capturing():
                gc.collect()
            return forward(*a, **k)

        new.model.forward = collecting
        gc.enable()
        assert new.generate([[1, 2, 3]], max_tokens=4, ignore_eos=True) == want
        assert False in calls and gc.isenabled() and new.runner.graph_captures == 1
    finally:
        gc.enable()
        gc.set_threshold(*was)
