"""The memory that the attention behind shared prefixes asks for."""
import pytest

from attention_kernel_triton_b200 import _lib


def sizes(tokens, heads, D, batch, groups):
    a = _lib.PrefixPagedArgs()
    c = a.chunk
    c.batch, c.num_tokens, c.num_qo_heads, c.num_kv_heads, c.page_size, c.head_dim = batch, tokens, heads, heads // 8, 16, D
    c.num_page_entries = 4096
    a.num_groups = groups
    return _lib.lib().akt_prefix_paged_workspace_size(a), _lib.lib().akt_chunk_paged_workspace_size(c)


@pytest.mark.parametrize("tokens,heads,D,batch", [(8192, 64, 128, 8), (500, 8, 64, 300), (1, 8, 128, 1)])
def test_no_results_of_rows_without_groups(tokens, heads, D, batch):
    # what the chunk attention takes, a place for each row of either kind, and tables of a few hundred bytes a sequence
    size, plain = sizes(tokens, heads, D, batch, 0)
    assert size <= plain + 16 * tokens * heads + 256 * batch + 16384
    # with groups, both results of every row
    size, _ = sizes(tokens, heads, D, batch, 1)
    assert size >= 8 * tokens * heads * D
