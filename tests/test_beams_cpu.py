"""Beam search's operators without a GPU: sizes, and refusals that come before any launch."""
import pytest
import torch


def test_sizes():
    from transformer_surgeon_b200 import _lib
    lib = _lib.load()
    assert [lib.tsb200_kv_record_bytes(_lib.KV_FP8_PAGE, d) for d in (64, 128)] == [16 * 64 + 16, 16 * 128 + 16]
    small, large = (lib.tsb200_beam_select_workspace_bytes(b, 4, 128256, _lib.BF16, 8) for b in (1, 64))
    assert 0 < small < large
    assert lib.tsb200_beam_select_workspace_bytes(0, 4, 128256, _lib.BF16, 8) == 0


def test_refusals_before_a_launch():
    from transformer_surgeon_b200 import ops
    scores = torch.zeros(2, 3)
    with pytest.raises(ValueError, match="CUDA"):
        ops.beam_select(torch.zeros(6, 10), scores)
    with pytest.raises(ValueError):
        ops.BeamReorder([])
    table, lens = torch.arange(4, dtype=torch.int32).reshape(2, 2), torch.zeros(2, dtype=torch.int32)
    kv = ops.PagedKV("fp8_page", 4, 1, 64, table, lens, "cpu")
    assert kv.k_scale is None and kv.fp8_scales_set
    with pytest.raises(ValueError, match="CUDA"):
        ops.BeamReorder([kv])
    with pytest.raises(ValueError):
        ops.BeamReorder([kv, ops.PagedKV("int8", 4, 1, 64, table, lens, "cpu")])
    with pytest.raises(ValueError, match="k_pool"):
        ops.PagedKV("fp8_page", 4, 1, 64, table, lens, "cpu", k_pool=torch.zeros(4, 1, 1024, dtype=torch.uint8))


def test_cache_vocabulary():
    from transformer_surgeon_b200 import blocks_path
    assert blocks_path.kv_format_of("paged_fp8_page") == "fp8_page"


def test_searches_that_selection_or_reordering_refuses_end_before_the_prompt():
    import types
    from transformer_surgeon_b200.decoder import CompressedDecoder

    def engine(rows):
        dec = CompressedDecoder.__new__(CompressedDecoder)
        dec.device, dec.B, dec.greedy_head, dec.max_seq_len, dec.cfg = "cpu", rows, False, 64, types.SimpleNamespace(vocab=100)

        def prefill(ids, beams):
            raise AssertionError("the prompt ran")
        dec.prefill = prefill
        return dec
    for rows, prompts, beams, kw in ((33, 1, 33, {}), (2080, 65, 32, {}), (4, 1, 4, dict(eos_token_id=7, pad_token_id=100)), (4, 1, 4, dict(eos_token_id=7, pad_token_id=-1)),
                                     (4, 1, 4, dict(eos_token_id=-1)), (4, 1, 3, {}), (4, 1, 0, {})):
        with pytest.raises(ValueError):
            engine(rows).beam_search(torch.zeros(prompts, 5, dtype=torch.int64), 5, beams, **kw)
    for rows, prompts, beams, kw in ((32, 1, 32, {}), (2048, 64, 32, {}), (4, 1, 4, dict(eos_token_id=7, pad_token_id=99)), (4, 1, 4, dict(pad_token_id=200))):
        with pytest.raises(AssertionError, match="the prompt ran"):
            engine(rows).beam_search(torch.zeros(prompts, 5, dtype=torch.int64), 5, beams, **kw)


class Elsewhere(torch.Tensor):
    """A CPU tensor that says it is on cuda:1, or wherever `at` says."""
    at = 1
    is_cuda = property(lambda self: self.at >= 0)
    device = property(lambda self: torch.device("cuda", self.at) if self.at >= 0 else torch.device("cpu"))

    def get_device(self):
        return self.at


class Here(Elsewhere):
    at = 0


@pytest.mark.parametrize("where", [Elsewhere, torch.Tensor])
def test_tensors_of_another_device_are_refused(monkeypatch, where):
    """One tensor of a call on another device than the current one (or on the host), the others there: refused before anything is launched."""
    from transformer_surgeon_b200 import ops
    monkeypatch.setattr(ops, "_current_device", lambda: 0)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_capturing", lambda: False)
    launched = []
    lib = ops._lib.load()

    class Library:
        def __getattr__(self, name):
            if name.endswith("_bytes"):
                return getattr(lib, name)
            return lambda *args: launched.append(name) or 0
    monkeypatch.setattr(ops._lib, "load", Library)

    def tensors(**shapes):
        return {k: torch.zeros(s, dtype=dt).as_subclass(Here) for k, (s, dt) in shapes.items()}

    def each_elsewhere(args, call):
        call(**args)
        assert launched.pop() and not launched
        for name in args:
            with pytest.raises(ValueError):
                call(**{**args, name: args[name].as_subclass(where)})
            assert not launched, name
    f32, i32, i64, u8 = torch.float32, torch.int32, torch.int64, torch.uint8
    each_elsewhere(tensors(logits=((4, 50), f32), scores=((2, 2), f32), finished=((2, 2), torch.bool), ws=((1 << 20,), u8), v=((2, 2), f32), p=((2, 2), i32), t=((2, 2), i64)),
                   lambda v, p, t, **kw: ops.beam_select(out=(v, p, t), **kw))
    kv = ops.PagedKV("fp8_page", 4, 1, 64, torch.arange(4, dtype=i32).reshape(2, 2).as_subclass(Here), torch.zeros(2, dtype=i32).as_subclass(Here), "cpu")
    kv.k_pool, kv.v_pool = kv.k_pool.as_subclass(Here), kv.v_pool.as_subclass(Here)
    each_elsewhere(tensors(q=((2, 2, 64), f32), out=((2, 2, 64), f32), ws=((1 << 20,), u8), seq_lens=((2,), i32)),
                   lambda q, **kw: ops.paged_decode_attention(kv, q, 32, **kw))
    each_elsewhere(tensors(k=((2, 1, 1, 64), f32), v=((2, 1, 1, 64), f32), new_lens=((2,), i32), seq_lens=((2,), i32)), kv.append)
    each_elsewhere(tensors(q=((2, 1, 2, 64), f32), k=((2, 1, 1, 64), f32), v=((2, 1, 1, 64), f32), cos=((8, 32), f32), sin=((8, 32), f32)),
                   lambda cos, sin, **kw: kv.rope_append(rope=(cos, sin), **kw))
    reorder = ops.BeamReorder.__new__(ops.BeamReorder)
    reorder.block_table, reorder.seq_lens, reorder.pages = kv.block_table, kv.seq_lens, ops.RowPages(kv.block_table)
    reorder._n, reorder._pools, reorder._scales = (2, 64, 4, 0, 1), torch.zeros(2, dtype=i64), None
    each_elsewhere(tensors(parents=((2,), i32), seq_lens=((2,), i32)), reorder)
    with pytest.raises(ValueError, match="uint8"):
        ops.beam_select(torch.zeros(4, 50).as_subclass(Here), torch.zeros(2, 2).as_subclass(Here), ws=torch.zeros(1 << 18, dtype=i32).as_subclass(Here))
    broken = ops.PagedKV("fp8_page", 4, 1, 64, kv.block_table, kv.seq_lens, "cpu", k_pool=kv.k_pool, v_pool=kv.v_pool.as_subclass(where) if where is Elsewhere else None)
    with pytest.raises(ValueError):
        ops.BeamReorder([broken])
    assert broken.pages is None and not launched
