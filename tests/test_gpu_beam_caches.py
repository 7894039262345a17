"""Caches that the caller owns, before, during and after a beam search: binding others, starting anew, setting back."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def wrapper_for(batch, kv_format="fp32", max_len=64):
    """A blocks-path wrapper over a tiny Llama of 512 tokens, and a model of the same weights."""
    from tests.test_gpu_hf import tiny
    from transformer_surgeon_b200 import blocks_path, surgeon
    model = tiny("llama", torch.float32)
    dec = surgeon.decoder_from_model(model, batch, max_len, kv_format)
    decoder = blocks_path.PagedTransformerDecoder(dec.cfg, dec.layers, dec.final_norm, "paged_" + kv_format, max_len, batch, dec.device)
    return blocks_path.LLMWrapper(model.get_input_embeddings(), decoder, model.lm_head)


def prompt(B, T, seed=5):
    return torch.randint(0, 512, (B, T), generator=torch.Generator().manual_seed(seed)).cuda()


def own(caches):
    return len(set(caches.block_table.flatten().tolist())) == caches.block_table.numel()


def close(a, b):
    """fp32 sums in other orders: products of 128 and 256 terms in a few layers, 2^-12 of the largest is far above them and far below another token's."""
    return (a - b).abs().max() <= 2.0 ** -12 * b.abs().max()


@pytest.mark.parametrize("kv_format", ["fp32", "fp8_page"])
def test_caches_leave_and_come_back_with_shared_pages(cuda, kv_format):
    """prefill(beams=3) on caches A, a prompt on B, and A again: A's rows still hold their prompts."""
    from transformer_surgeon_b200 import blocks_path
    w = wrapper_for(6, kv_format)
    a, b = (blocks_path.build_paged_caches(w.decoder) for _ in range(2))
    ids = prompt(2, 37)
    w._bind(a)
    w.engine.prefill(ids, beams=3)
    table, tokens = a.block_table.clone(), prompt(6, 1, 6)
    assert not own(a)
    w.prefill(prompt(6, 11, 7), b)
    assert torch.equal(a.block_table, table) and own(b)
    got = w(tokens, torch.tensor([37]), a)[0].clone()
    straight = wrapper_for(6, kv_format)
    c = blocks_path.build_paged_caches(straight.decoder)
    straight._bind(c)
    straight.engine.prefill(ids, beams=3)
    assert torch.equal(got, straight(tokens, torch.tensor([37]), c)[0])
    # a search on the caches that came back, and on those that left
    for caches, engine in ((a, w), (b, w)):
        engine._bind(caches)
        seqs, scores = engine.engine.beam_search(ids, 8, 3)
        straight._bind(c)
        want = straight.engine.beam_search(ids, 8, 3)
        assert torch.equal(seqs, want[0]) and torch.equal(scores, want[1])


def test_another_engine_takes_over_shared_pages(cuda):
    """Caches searched by one engine, bound to a second: it knows the rows' own pages too."""
    from transformer_surgeon_b200 import blocks_path
    w, other = wrapper_for(6), wrapper_for(6)
    caches, ids = blocks_path.build_paged_caches(w.decoder), prompt(2, 37)
    w._bind(caches)
    want = w.engine.beam_search(ids, 8, 3)
    assert not own(caches)
    other._bind(caches)
    got = other.engine.beam_search(ids, 8, 3)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    other.engine.reset()
    assert own(caches) and int(caches.seq_lens.max()) == 0


@pytest.mark.parametrize("how", ["beam_search", "prefill"])
def test_caches_reset_after_beams(cuda, how):
    """PagedCaches.reset: every row its own pages again, so that tokens one by one are what they are on new caches."""
    from transformer_surgeon_b200 import blocks_path
    w = wrapper_for(6, "fp8_page")
    caches, fresh = (blocks_path.build_paged_caches(w.decoder) for _ in range(2))
    w._bind(caches)
    if how == "beam_search":
        w.engine.beam_search(prompt(2, 19), 20, 3)
    else:
        w.engine.prefill(prompt(2, 37), beams=3)
    assert not own(caches)
    caches.reset()
    assert own(caches) and int(caches.seq_lens.max()) == 0        # before anything is appended: rows that share a page would write it at once
    ids, got = prompt(6, 21, 8), []
    for t in range(21):
        got.append(w(ids[:, t], torch.tensor([t]), caches)[0].clone())
    for t in range(21):
        assert torch.equal(got[t], w(ids[:, t], torch.tensor([t]), fresh)[0])


@pytest.mark.parametrize("captured", [False, True])
def test_caches_hold_the_sequences_that_a_search_returns(cuda, captured):
    """After beam_search, row by row: the next step goes on from the returned sequence, not from the beams ahead of the last selection."""
    from tests.test_gpu_hf import tiny
    from transformer_surgeon_b200 import surgeon
    model = tiny("llama", torch.float32)
    dec, alone = (surgeon.decoder_from_model(model, 6, 64, "fp32") for _ in range(2))
    if captured:
        dec.capture()
    for T, new in ((19, 30), (19, 29), (16, 1), (37, 8), (9, 8)):
        seqs, _ = dec.beam_search(prompt(2, T, T + new), new, 3)
        rows = torch.cat((seqs.flatten(0, 1), prompt(6, 3, 9)), 1)
        alone.reset()
        for t in range(T + new - 1):
            alone.step(rows[:, t])
        assert torch.equal(dec.seq_lens, alone.seq_lens)
        for t in range(T + new - 1, rows.shape[1]):
            assert close(dec.step(rows[:, t]), alone.step(rows[:, t]))


@pytest.mark.parametrize("pos", [0, 5, 16, 30, 47])
def test_steps_set_back_after_a_search(cuda, pos):
    """`forward` at any position after a beam search, which it accepts as the blocks path does: every row goes on from its own sequence's first tokens."""
    from transformer_surgeon_b200 import blocks_path
    w, B, K, T, new = wrapper_for(6), 2, 3, 19, 30
    caches, fresh = (blocks_path.build_paged_caches(w.decoder) for _ in range(2))
    w._bind(caches)
    seqs, _ = w.engine.beam_search(prompt(B, T), new, K)
    rows = seqs.flatten(0, 1)                                      # 48 of their 49 tokens are cached
    after, got = prompt(6, 3, 9), []
    for t in range(3):
        got.append(w(after[:, t], torch.tensor([pos + t]), caches)[0].clone())
    assert own(caches) or pos >= 48 // 16 * 16
    for t in range(pos):
        w(rows[:, t], torch.tensor([t]), fresh)
    for t in range(3):
        assert close(got[t], w(after[:, t], torch.tensor([pos + t]), fresh)[0])


def test_steps_that_go_on_after_a_search(cuda):
    """Positions behind the search: the pages stay shared, and every row goes on from its whole sequence."""
    from transformer_surgeon_b200 import blocks_path
    w = wrapper_for(6)
    caches, fresh = (blocks_path.build_paged_caches(w.decoder) for _ in range(2))
    w._bind(caches)
    seqs, _ = w.engine.beam_search(prompt(2, 37), 8, 3)
    rows, got = torch.cat((seqs.flatten(0, 1), prompt(6, 6, 9)), 1), []
    for t in range(44, rows.shape[1]):
        got.append(w(rows[:, t], torch.tensor([t]), caches)[0].clone())
    assert not own(caches)
    for t in range(rows.shape[1]):
        logits = w(rows[:, t], torch.tensor([t]), fresh)[0]
        assert t < 44 or close(got[t - 44], logits)


def test_a_captured_reordering_is_never_taken_for_the_last_one(cuda):
    """A graph of a reordering, replayed behind a reset: a step that sets sequences back still finds that rows share pages."""
    from transformer_surgeon_b200 import blocks_path, ops
    w = wrapper_for(6)
    caches = blocks_path.build_paged_caches(w.decoder)
    reorder = ops.BeamReorder(caches.kv)
    parents = torch.tensor([0, 0, 0, 3, 3, 3], dtype=torch.int32, device=cuda)
    graph = torch.cuda.CUDAGraph()
    reorder(parents)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        reorder(parents)
    caches.reset()
    ids = prompt(6, 37)
    want = w.prefill(ids, caches)[0].clone()
    graph.replay()
    assert not own(caches)
    got = w(ids[:, 10], torch.tensor([10]), caches)[0].clone()
    assert own(caches)
    w.prefill(ids[[0, 0, 0, 3, 3, 3]], caches)
    assert close(got, w(ids[:, 10], torch.tensor([10]), caches)[0])
    assert torch.equal(w.prefill(ids, caches)[0], want)
