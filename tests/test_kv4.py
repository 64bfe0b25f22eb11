"""What the operators of a cache held in 4 bits refuse, before anything reaches a GPU."""
import pytest
import torch

BF16, I32 = torch.bfloat16, torch.int32


@pytest.fixture
def ops():
    from binfer_b200.csrc import ops
    return ops


def _i(*shape):
    return torch.zeros(shape, dtype=I32)


def test_cache_layout(ops):
    c = ops.kv4_cache(5, 2, 16, 128, "cpu")
    assert tuple(c.shape) == (5, 2, 2, 1152) and c.dtype == torch.uint8 and not c.any()
    assert ops.kv4_takes(BF16, 128, 16) and not ops.kv4_takes(torch.float32, 128, 16)
    for d, ps in ((96, 16), (32, 16), (128, 4), (128, 24), (128, 256), (128, 17)):
        assert not ops.kv4_takes(BF16, d, ps)
        with pytest.raises(ops.KernelError):
            ops.kv4_cache(5, 2, ps, d, "cpu")
    for pages, heads in ((0, 1), (1, 0)):
        with pytest.raises(ops.KernelError):
            ops.kv4_cache(pages, heads, 16, 128, "cpu")


def test_no_cpu_path(ops):
    c, k = ops.kv4_cache(3, 1, 16, 64, "cpu"), torch.zeros((2, 64), dtype=BF16)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.kv4_store(k, k, _i(2), c, _i(1))
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.kv4_load(c, _i(1, 2), _i(1, 4), 1, 64, _i(1))
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.kv4_decode_attention(k, c, None, 2, _i(2), _i(2), _i(1, 2), k, 1, 1, 64, None, 1.0, _i(1))
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.kv4_prefill_attention(k, c, _i(1, 4), 1, 2, _i(1, 2), k, 1, 1, 64, None, 1.0, _i(1), 64, 2)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.step_tables(_i(2, 4), _i(1, 5), _i(1), 16, 8, _i(2), _i(1), _i(1), _i(1), _i(1), _i(1, 4), _i(1))


def _store_args(ops):
    return dict(k=torch.zeros((2, 128), dtype=BF16), v=torch.zeros((2, 128), dtype=BF16), slots=_i(2),
                cache=ops.kv4_cache(3, 2, 16, 64, "cpu"), err=_i(1))


@pytest.mark.parametrize("change", [dict(k=torch.zeros((2, 128))), dict(v=torch.zeros((3, 128), dtype=BF16)),
                                    dict(k=torch.zeros((128, 2), dtype=BF16).T), dict(slots=_i(2).long()),
                                    dict(k=torch.zeros((2, 2, 64), dtype=BF16)), dict(err=torch.zeros(1)),
                                    dict(cache=torch.zeros((3, 2, 2, 576), dtype=torch.int8)),
                                    dict(cache=torch.zeros((3, 2, 2, 575), dtype=torch.uint8)),
                                    dict(cache=torch.zeros((3, 2, 3, 576), dtype=torch.uint8)),
                                    dict(cache=torch.zeros((6, 2, 576), dtype=torch.uint8)),
                                    dict(cache=torch.zeros((3, 2, 4, 576), dtype=torch.uint8)[:, :, ::2])])
def test_store_refuses(ops, change):
    with pytest.raises(ops.KernelError) as e:
        ops.kv4_store(**dict(_store_args(ops), **change))
    assert "CPU path" not in str(e.value)


def _attention_args(ops):
    q = torch.zeros((3, 256), dtype=BF16)
    return dict(q=q, cache=ops.kv4_cache(3, 2, 16, 64, "cpu"), block_tables=_i(2, 4), out=torch.zeros_like(q),
                nh=4, nkv=2, d=64, window=None, scale=0.1, err=_i(1))


@pytest.mark.parametrize("change", [dict(block_tables=_i(2, 4).long()), dict(block_tables=_i(8)),
                                    dict(block_tables=_i(4, 2).T), dict(err=torch.zeros(1, dtype=torch.int64))])
def test_attention_refuses(ops, change):
    args = dict(_attention_args(ops), **change)
    decode = dict(rows=None, n_rows=3, seq_of_token=_i(3), positions=_i(3))
    with pytest.raises(ops.KernelError) as e:
        ops.kv4_decode_attention(**args, **decode)
    assert "CPU path" not in str(e.value)
    with pytest.raises(ops.KernelError) as e:
        ops.kv4_prefill_attention(**args, items=_i(1, 4), n_items=1, max_rows=3, ctx_rows=64, max_ctx=3)
    assert "CPU path" not in str(e.value)


@pytest.mark.parametrize("change", [dict(seq_of_token=_i(3).long()), dict(positions=torch.zeros(3)),
                                    dict(rows=torch.zeros(3))])
def test_decode_attention_refuses(ops, change):
    args = dict(_attention_args(ops), rows=None, n_rows=3, seq_of_token=_i(3), positions=_i(3))
    with pytest.raises(ops.KernelError, match="must be"):
        ops.kv4_decode_attention(**dict(args, **change))


def test_items_are_int32(ops):
    with pytest.raises(ops.KernelError, match="items"):
        ops.kv4_prefill_attention(**_attention_args(ops), items=_i(1, 4).long(), n_items=1, max_rows=3, ctx_rows=64,
                                  max_ctx=3)
    with pytest.raises(ops.KernelError, match="items"):
        ops.kv4_load(ops.kv4_cache(3, 1, 16, 64, "cpu"), _i(1, 2), torch.zeros((1, 4)), 1, 64, _i(1))


@pytest.mark.parametrize("name", ["master", "entries", "new_pages", "q_start", "positions", "seq_of_token",
                                  "ctx_lens", "slots", "tables", "err", "decode_rows", "prefill_items"])
def test_step_tables_takes_int32(ops, name):
    args = dict(master=_i(2, 4), entries=_i(1, 5), new_pages=_i(1), page_size=16, num_pages=8, q_start=_i(2),
                positions=_i(1), seq_of_token=_i(1), ctx_lens=_i(1), slots=_i(1), tables=_i(1, 4), err=_i(1),
                decode_rows=_i(1), prefill_items=_i(0, 4))
    args[name] = args[name].long()
    with pytest.raises(ops.KernelError, match="int32"):
        ops.step_tables(**args)


@pytest.mark.parametrize("change", [dict(variant="fast"), dict(variant="load", q=torch.zeros((3, 512), dtype=BF16)[:, :256]),
                                    dict(variant="load", scale=0.0)])
def test_prefill_variants(ops, change, monkeypatch):
    """(The checks before a launch, with the device's left out.)"""
    monkeypatch.setattr(ops, "_same_device", lambda *a: None)
    args = dict(_attention_args(ops), items=_i(1, 4), n_items=1, max_rows=3, ctx_rows=64, max_ctx=3)
    with pytest.raises(ops.KernelError, match="variant"):
        ops.kv4_prefill_attention(**dict(args, **change))


@pytest.mark.parametrize("what,change", [
    ("window", dict(window=0)), ("keep_first", dict(keep_first=-1)), ("heads", dict(nkv=1)), ("heads", dict(d=128)),
    ("heads", dict(nh=3)), ("q", dict(q=torch.zeros((3, 256)))), ("q", dict(q=torch.zeros((3, 512), dtype=BF16)[:, 1:257])),
    ("tokens", dict(block_tables=_i(1, (1 << 20) + 1))), ("out", dict(out=torch.zeros((3, 255), dtype=BF16))), ("out", dict(out=torch.zeros((2, 256), dtype=BF16)))])
def test_attention_sizes(ops, what, change, monkeypatch):
    monkeypatch.setattr(ops, "_same_device", lambda *a: None)
    args = dict(_attention_args(ops), **change)
    with pytest.raises(ops.KernelError, match=what):
        ops.kv4_decode_attention(**args, rows=None, n_rows=3, seq_of_token=_i(3), positions=_i(3))
    with pytest.raises(ops.KernelError, match=what):
        ops.kv4_prefill_attention(**args, items=_i(1, 4), n_items=1, max_rows=3, ctx_rows=64, max_ctx=3)


@pytest.mark.parametrize("change", [dict(n_rows=4), dict(n_rows=-1), dict(rows=_i(2)), dict(seq_of_token=_i(2)),
                                    dict(positions=_i(2))])
def test_decode_rows(ops, change, monkeypatch):
    monkeypatch.setattr(ops, "_same_device", lambda *a: None)
    args = dict(_attention_args(ops), rows=None, n_rows=3, seq_of_token=_i(3), positions=_i(3))
    with pytest.raises(ops.KernelError, match="rows inside q"):
        ops.kv4_decode_attention(**dict(args, **change))


@pytest.mark.parametrize("change", [dict(n_items=2), dict(n_items=-1), dict(ctx_rows=65), dict(max_rows=-1)])
def test_prefill_items(ops, change, monkeypatch):
    monkeypatch.setattr(ops, "_same_device", lambda *a: None)
    args = dict(_attention_args(ops), items=_i(1, 4), n_items=1, max_rows=3, ctx_rows=64, max_ctx=3)
    with pytest.raises(ops.KernelError, match="items"):
        ops.kv4_prefill_attention(**dict(args, **change))


@pytest.mark.parametrize("change", [dict(rows=63), dict(rows=0), dict(n_items=0), dict(n_items=2), dict(items_out=_i(3)),
                                    dict(window=0), dict(places=-1)])
def test_load_sizes(ops, change, monkeypatch):
    monkeypatch.setattr(ops, "_same_device", lambda *a: None)
    args = dict(cache=ops.kv4_cache(3, 1, 16, 64, "cpu"), block_tables=_i(1, 2), items=_i(1, 4), n_items=1, rows=64,
                err=_i(1))
    with pytest.raises(ops.KernelError):
        ops.kv4_load(**dict(args, **change))


@pytest.mark.parametrize("change", [dict(entries=_i(1, 4)), dict(page_size=0), dict(num_pages=0), dict(tables=_i(0, 4)),
                                    dict(q_start=_i(1)), dict(ctx_lens=_i(0)), dict(num_pages=1 << 28)])
def test_step_tables_sizes(ops, change, monkeypatch):
    monkeypatch.setattr(ops, "_same_device", lambda *a: None)
    args = dict(master=_i(2, 4), entries=_i(1, 5), new_pages=_i(1), page_size=16, num_pages=8, q_start=_i(2),
                positions=_i(1), seq_of_token=_i(1), ctx_lens=_i(1), slots=_i(1), tables=_i(1, 4), err=_i(1))
    with pytest.raises(ops.KernelError, match="step_tables"):
        ops.step_tables(**dict(args, **change))


def test_which_portions_are_loaded(ops):
    """The rule's two sides at sizes where they are far apart."""
    pays = ops._kv4_load_pays
    assert pays(1, 2048, 2048, 0, 0, 32, 8, 128) and pays(1, 256, 8448, 0, 0, 32, 8, 128)
    assert not pays(6, 5, 3005, 0, 0, 16, 8, 128) and not pays(1, 128, 1128, 0, 0, 32, 8, 128)
    assert pays(1, 1024, 5024, 0, 0, 16, 4, 64) and not pays(1, 256, 1256, 0, 0, 16, 4, 64)
    assert pays(1, 1024, 5024, 0, 0, 8, 2, 256) and not pays(1, 64, 1064, 0, 0, 8, 2, 256)
    assert pays(1, 1024, 100000, 512, 0, 32, 8, 128) and not pays(1, 8, 100000, 0, 0, 32, 8, 128)


def test_numbers_that_an_argument_has_no_room_for():
    from binfer_b200.csrc import ops
    with pytest.raises(ops.KernelError, match="no room"):
        ops._Packed("bf_kv4_store", "i")(1 << 40)


@pytest.mark.parametrize("change", [dict(nkv=1), dict(d=64), dict(nh=3), dict(qkv=torch.zeros((3, 1024))),
                                    dict(qkv=torch.zeros((3, 2048), dtype=BF16)[:, ::2]), dict(slots=_i(2)), dict(positions=_i(2)),
                                    dict(q_w=torch.zeros(64)), dict(inv_freq=torch.zeros(65)), dict(k_w=torch.zeros(128, dtype=BF16)),
                                    dict(q_out=torch.zeros((3, 256), dtype=BF16)), dict(slots=torch.zeros(3))])
def test_norm_rotation_and_store_refusals(ops, change, monkeypatch):
    monkeypatch.setattr(ops, "_same_device", lambda *a: None)
    args = dict(qkv=torch.zeros((3, 1024), dtype=BF16), q_w=torch.zeros(128), k_w=torch.zeros(128), inv_freq=torch.zeros(64),
                positions=_i(3), slots=_i(3), q_out=torch.zeros((3, 512), dtype=BF16),
                cache=torch.zeros((2, 2, 2, 1152), dtype=torch.uint8), nh=4, nkv=2, d=128, eps=1e-6, err=_i(1))
    with pytest.raises(ops.KernelError):
        ops.qk_norm_rope_kv4_store(**dict(args, **change))
