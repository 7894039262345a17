"""Caches that beams shared, without a GPU: what `reset` and a step that sets sequences back do to the block table and the pages."""
import torch


def caches_on_cpu(fmt="fp8_page"):
    from transformer_surgeon_b200 import blocks_path, ops
    table, lens = torch.arange(12, dtype=torch.int32).reshape(3, 4), torch.full((3,), 40, dtype=torch.int32)
    kv = [ops.PagedKV(fmt, 12, 1, 64, table, lens, "cpu") for _ in range(2)]
    for i, x in enumerate(kv):
        x.pages = kv[0].pages or ops.RowPages(table)
        for side, pool in enumerate((x.k_pool, x.v_pool)):
            pool.copy_((torch.arange(12) + 100 * side + 50 * i)[:, None, None].expand_as(pool))
    return blocks_path.PagedCaches(kv, table, lens, "paged_" + fmt)


def share(caches):
    """What a reordering with parents [1, 1, 0] does to the full pages at a length of 40."""
    home = caches.block_table.clone()
    caches.block_table[:, :2] = home[[1, 1, 0], :2]
    caches.kv[0].pages.shared = True
    return home


def test_reset_gives_rows_their_own_pages():
    caches = caches_on_cpu()
    home = share(caches)
    caches.reset()
    assert torch.equal(caches.block_table, home) and not caches.seq_lens.any() and not caches.kv[0].pages.shared


def test_a_step_that_sets_sequences_back_separates_their_pages():
    """A position in the open page or behind it changes nothing; one below copies what rows share into their own pages."""
    import types
    from transformer_surgeon_b200 import blocks_path
    caches = caches_on_cpu()
    home = share(caches)
    shared, before = caches.block_table.clone(), [p.clone() for x in caches.kv for p in (x.k_pool, x.v_pool)]
    w = blocks_path.LLMWrapper.__new__(blocks_path.LLMWrapper)
    w.engine = types.SimpleNamespace(device="cpu", B=3, cfg=types.SimpleNamespace(kv_format="fp8_page"), step=lambda tokens: torch.zeros(3, 5))
    w.decoder, w.cache_impl, w._bound = types.SimpleNamespace(max_cache_len=64), caches.cache_impl, caches
    for pos in (40, 41, 32):
        w(torch.zeros(3, dtype=torch.int64), torch.tensor([pos]), caches)
        assert torch.equal(caches.block_table, shared)
    caches.seq_lens.fill_(40)
    w(torch.zeros(3, dtype=torch.int64), torch.tensor([31]), caches)
    assert torch.equal(caches.block_table, home) and not caches.kv[0].pages.shared and caches.seq_lens.tolist() == [31] * 3
    for pool, old in zip([p for x in caches.kv for p in (x.k_pool, x.v_pool)], before):
        for row in range(3):
            for page in range(4):
                assert torch.equal(pool[home[row, page]], old[shared[row, page]])


def test_reset_leaves_a_table_alone_that_no_beams_share():
    """Pages handed out anew by the caller, after a search was over and put back: a reset does not take them away."""
    caches = caches_on_cpu()
    share(caches)
    caches.reset()
    mine = caches.block_table.flip(0).clone()
    caches.block_table.copy_(mine)
    caches.reset()
    assert torch.equal(caches.block_table, mine)
