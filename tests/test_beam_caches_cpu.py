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
