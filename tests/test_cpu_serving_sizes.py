"""Sizes whose products pass 64 bits: refused before anything is launched, on a host
without a GPU."""
from test_cpu_serving import paged, pytestmark, refused, seqs, tree  # noqa: F401


def test_tree_grids_beyond_64_bits():
    """2^56 workgroups of 256 threads: 2^64 of them, 0 in 64 bits."""
    refused("more rows than one launch covers", paged(kv_heads=1).tree_attention_workspace,
            seqs(batch=1 << 30, stride=1 << 20, most=1 << 15),
            tree(batch=1 << 30, most=1024, total=1000, mask_stride=32), 1 << 20)
    kv = paged(kv_heads=1 << 26, head_dim=8)
    refused("more rows than one launch covers", kv.tree_attention_workspace,
            seqs(batch=1 << 30), tree(batch=1 << 30, most=1), 1 << 26)
