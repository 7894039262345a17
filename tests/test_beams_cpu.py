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
