"""Sizes whose products pass 64 bits, or ranks that pass 32: refused before anything is
launched, on a host without a GPU."""
from test_cpu_serving import (At, paged, pool, pytestmark, reaches, refused, reorder,  # noqa: F401
                              seqs, table, tree)


def test_tree_grids_beyond_64_bits():
    """2^56 workgroups of 256 threads: 2^64 of them, 0 in 64 bits."""
    refused("more rows than one launch covers", paged(kv_heads=1).tree_attention_workspace,
            seqs(batch=1 << 30, stride=1 << 20, most=1 << 15),
            tree(batch=1 << 30, most=1024, total=1000, mask_stride=32), 1 << 20)
    kv = paged(kv_heads=1 << 26, head_dim=8)
    refused("more rows than one launch covers", kv.tree_attention_workspace,
            seqs(batch=1 << 30), tree(batch=1 << 30, most=1), 1 << 26)


def test_tables_whose_entries_pass_32_bits():
    """Fresh pages are numbered over all entries of the new table."""
    base, wide = 1 << 40, 1 << 16
    new = dict(stride=wide, lengths=At(1 << 28), held=At(1 << 29))
    p = pool(pages=1000)
    refused("invalid table", reorder, p, None, table(base, batch=wide, **new))
    refused("invalid table", p.reorder_workspace, table(), table(base, batch=wide, **new))
    reaches(reorder, p, None, table(base, batch=wide - 1, **new), copies=At(1 << 34))
    reaches(reorder, p, table(base, batch=wide, **new), None)
